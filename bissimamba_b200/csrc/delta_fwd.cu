// delta_fwd.cu -- gated delta rule, forward recurrence over chunks
// (kmb_delta.cuh: a unit of 16 columns of dv, four warps):
//   X = V - e^gamma K S;  W = M X;  U = beta W;  O = scale (e^gamma Q S + P U);  S <- e^gamma_C S + K^T (G_C. U)
// all transposed.  The chain of a chunk is latency: three products that each wait
// for the last, with fp16 pieces made and passed on between them.  So all fragments
// of a product are loaded before its first instruction, blocks alternate in the
// tensor cores, and what is not the chain is the side warps'.  These have two
// pieces of every fp32 factor too (o is rounded once, whether or not the backward
// follows): their products share the tensor cores with the chain's, so blocks above
// the diagonal are left out there (long prompt 615 -> 592 us).
// Measured (16384 tokens, 16 heads of 128, bf16): 484 us, 1.89 us a chunk, of which one
// piece in the side warps' products would save 0.14; one warp for all of dk took
// 6.5 us, four warps with everything in them 2.1 us.
#include "kmb_delta.cuh"
#include "kmb_launch.cuh"

namespace kmb {
namespace {

template <int DKP, typename IO>
struct FwdSmem {
    static constexpr int C = kDeltaC;
    static constexpr int NPK = sizeof(IO) == 4 ? 2 : 1;
    using ST = DeltaStage<C, DKP, NPK>;
    using FS = FragBuf<DKP / 16, 2>;
    using FX = FragBuf<C / 16, 2>;
    // of a unit: fragments of S, X, G_C. U and U, W as accumulators
    static constexpr int SW = FS::BYTES + 4096, XUO = 3 * FX::BYTES;
    // Where two stages of K, Q and M, three of P and the token factors and two buffers of S and W fit, the side warps
    // finish a chunk's outputs during the next chunk (LAG), and only one barrier a chunk holds the chain to them.
    // Else two stages of all, and the chain waits for them between its own steps.
    static constexpr bool lag(int nu) {
        return 2 * ST::FRONT + 3 * ST::REAR + nu * (2 * SW + XUO) + nu * 2048 + 128 <= 227 * 1024;
    }
    static constexpr int rears(int nu) { return lag(nu) ? 3 : 2; }
    static constexpr int tiles(int nu) { return 2 * ST::FRONT + rears(nu) * ST::REAR; }
    static constexpr int ex(int nu) { return (lag(nu) ? 2 : 1) * SW + XUO; }
    static constexpr int bytes(int nu) { return tiles(nu) + nu * ex(nu); }
};

template <int DKP, typename IO, bool KEEP, int NU>
__global__ void __launch_bounds__(256 * NU, 1)
delta_chain_fwd_kernel(const __grid_constant__ DeltaDesc d, int vec) {
    using SM = FwdSmem<DKP, IO>;
    constexpr int C = kDeltaC, NPK = SM::NPK;
    using ST = typename SM::ST;
    using FS = typename SM::FS;
    using FX = typename SM::FX;
    constexpr int KT = DKP / 8, KTW = KT / 4, KBW = DKP / 64;   // dk tiles, of a warp; its blocks of 16
    constexpr int PK = C * DKP * 2;              // bytes of a K or Q piece
    extern __shared__ __align__(128) unsigned char sm[];
    constexpr int NS = SM::rears(NU);
    constexpr bool LAG = SM::lag(NU);
    __shared__ __align__(8) uint64_t full[NS];
    __shared__ __align__(16) unsigned char vbuf[NU * 4][512];
    const uint32_t sb = (uint32_t)__cvta_generic_to_shared(sm);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = warp >> 3, w = warp & 3;
    const bool chain = (warp & 4) == 0;
    unsigned char* ex = sm + SM::tiles(NU) + grp * SM::ex(NU);
    unsigned char *exX = ex, *exU = exX + FX::BYTES, *exO = exU + FX::BYTES;
    // buffers of step i
    const auto bufS = [&](int i) { return exO + FX::BYTES + (LAG ? (i & 1) * SM::SW : 0); };
    const auto bufW = [&](int i) { return bufS(i) + FS::BYTES; };
    const int ub = (d.units + NU - 1) / NU;
    const int u = (int)(blockIdx.x % ub) * NU + grp;
    const int hv = (int)(blockIdx.x / ub) % d.Hv, nr = (int)(blockIdx.x / ub) / d.Hv;
    pdl_release();
    pdl_wait();
    const int n = d.order ? d.order[nr] : nr;
    const bool on = u < d.units;                 // a unit past dv computes on zeros and stores nothing
    const int r = lane >> 2, c2 = (lane & 3) * 2;
    const int col[2] = {u * 16 + r, u * 16 + r + 8};
    const bool cok[2] = {col[0] < d.dv, col[1] < d.dv};
    const int ldv = (int)d.ld_v, ldo = (int)d.ld_o;
    long long start, len;
    seq_range(d, n, start, len);
    const int chunk0 = d.cu ? d.cstart[n] : n * d.nc;
    const int nch = (int)((len + C - 1) / C);
    const size_t sbase = ((size_t)n * d.Hv + hv) * d.dk * d.dv;

    // stages of step i's tiles (s: its P and token factors)
    const auto front = [&](int i) { return sb + (i & 1) * ST::FRONT; };
    const auto rear = [&](int s) { return sb + 2 * ST::FRONT + s * ST::REAR; };
    const auto factors = [&](int s) { return (const float*)(sm + 2 * ST::FRONT + s * ST::REAR + ST::oTok); };
    // the side warps of the first unit copy the tiles of the recurrence's step i into its stages
    const bool copies = warp >= 4 && warp < 8 && lane == 0;
    const auto fetch = [&](int i, int s) {
        ST::load(d, d.Mt, front(i), rear(s), smem_u32(&full[s]), chunk0 + i, hv, w);
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; i++) mbar_init(smem_u32(&full[i]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (copies && nch > 0) fetch(0, 0);
    // The chunk's tiles are there, the state's fragments too, and what the next step's tiles replace is read; false:
    // a wait ran out.
    int slot = 0, phase = 0, last_slot = 0;   // of the step's tiles, of the last step's
    const auto begin = [&](int i) {
        if (i > 0) {
            last_slot = slot;
            if (++slot == NS) {
                slot = 0;
                phase ^= 1;
            }
        }
        // The side warps wait for the copies; the barrier passes on what they saw, and all threads leave together.
        const bool got = chain || mbar_wait(smem_u32(&full[slot]), phase);
        if (!__syncthreads_and(got)) {
            if (!got) {
                set_status(d.status, KMB_ERR_TIMEOUT_FULL);
                mbar_wait(smem_u32(&full[slot]), phase);   // the block's memory stays its own for another limit
            }
            return false;
        }
        if (copies && i + 1 < nch) fetch(i + 1, slot + 1 == NS ? 0 : slot + 1);
        return true;
    };

    if (chain) {
        float S[KTW][4];
        // a reset at the first token forgets the initial state, whatever it holds (0 times an infinity or NaN would stay one)
        const bool carry = d.h0 && !(d.g && len > 0 && expf(d.g[start * d.Hv + hv]) == 0.0f);
#pragma unroll
        for (int t = 0; t < KTW; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = (w * KTW + t) * 8 + c2 + (e & 1);
                S[t][e] = (carry && i < d.dk && cok[e >> 1]) ? d.h0[sbase + (size_t)i * d.dv + col[e >> 1]] : 0.0f;
            }
        TokenTile<IO> Vn;   // v of the warp's tokens of the next chunk
        const auto load_v = [&](int c) {
            const long long t0 = (long long)c * C + w * 16;
            Vn.load(d.v, start + t0, ldv, (long long)hv * d.dv + u * 16, on ? d.dv - u * 16 : 0,
                    (int)(len - t0 < 16 ? len - t0 : 16), lane, vec);
        };
        const auto put_state = [&](int i) {   // for step i
            unsigned char* exS = bufS(i);
            if (KEEP && on && i < nch)
                put_acc((unsigned char*)(d.Sf + (((size_t)(chunk0 + i) * d.Hv + hv) * d.units + u) * 16 * DKP), w * KTW, lane, S);
            float up, dn;
            frag_scale(S, up, dn);
#pragma unroll
            for (int b = 0; b < KBW; b++) {
                uint32_t a[2][4];
                frag_pieces<2>(S[2 * b], S[2 * b + 1], up, a);
                FS::put(exS, w * KBW + b, lane, a, dn);
            }
        };
        put_state(0);
        __syncthreads();
        float V[2][4];
        if (nch > 0) load_v(0);
        for (int c = 0; c < nch; c++) {
            if (!begin(c)) return;
            Vn.tiles(V, vbuf[grp * 4 + w], lane, vec);
            if (c + 1 < nch) load_v(c + 1);
            const uint32_t st = front(c);
            const float* tk = factors(slot);
            const float* tw = tk + w * 16 + c2;      // factors of the warp's tokens
            const unsigned char* exS = bufS(c);
            float X[2][4], part[4][2][4], dn, up;
            zero(X);
#pragma unroll
            for (int k0 = 0; k0 < DKP / 16; k0 += 4) {
                mma_blocks<4, 2, NPK, 2>(
                    part, [&](int k, uint32_t (&a)[2][4]) { FS::template get<2>(exS, k0 + k, lane, a); },
                    [&](int k, int p, int, uint32_t (&f)[4]) {
                        ldm4(f, st + p * PK + wide_off<C>(w * 16 + lb_row(lane), (k0 + k) * 16 + lb_col(lane)));
                    });
#pragma unroll
                for (int k = 0; k < 4; k++) add_scaled(X, part[k], FS::scale(exS, k0 + k));
            }
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + (e & 1);
                    X[t][e] = V[t][e] - tw[TOK_EG * C + i] * tw[TOK_FK * C + i] * X[t][e];
                }
            frag_scale(X, up, dn);
            FX::put(exX, w, lane, X, up, dn);
            chain_bar(grp);
            // W^T = X M^T: row i of M reaches columns j <= i only
            float W[2][4];
            zero(W);
            const float fm = tk[TOK_MISC * C + w];
            mma_blocks<4, 2, 2, 2>(
                part, [&](int k, uint32_t (&a)[2][4]) { FX::template get<2>(exX, k, lane, a); },
                [&](int k, int p, int, uint32_t (&f)[4]) {
                    ldm4(f, st + ST::oT + p * ST::TT + tile_off<C>(w * 16 + lb_row(lane), k * 16 + lb_col(lane)));
                });
#pragma unroll
            for (int k = 0; k < 4; k++) add_masked(W, part[k], FX::scale(exX, k) * fm, k <= w ? ~0u : 0u);
            put_acc(bufW(c), w * 2, lane, W);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + (e & 1);
                    W[t][e] *= tw[TOK_BETA * C + i] * (tw[TOK_GC * C + i] * tw[TOK_FK * C + i]);
                }
            frag_scale(W, up, dn);
            FX::put(exU, w, lane, W, up, dn);
            if (LAG) chain_bar(grp);
            else unit_bar(grp);
            // S^T <- e^gamma_C S^T + (G_C. U)^T K
            const float last = tk[TOK_EG * C + C - 1];
#pragma unroll
            for (int t = 0; t < KTW; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) S[t][e] *= last;
            constexpr int KB = KTW == 2 || NU == 1 ? 4 : 2;   // blocks at a time: what registers allow
#pragma unroll
            for (int k0 = 0; k0 < C / 16; k0 += KB) {
                float ps[KB][KTW][4];
                mma_blocks<KB, 2, NPK, KTW>(
                    ps, [&](int k, uint32_t (&a)[2][4]) { FX::template get<2>(exU, k0 + k, lane, a); },
                    [&](int k, int p, int t2, uint32_t (&f)[4]) {
                        ldm4t(f, st + p * PK + wide_off<C>((k0 + k) * 16 + la_row(lane), (w * KTW + t2 * 2) * 8 + la_col(lane)));
                    });
#pragma unroll
                for (int k = 0; k < KB; k++) add_scaled(S, ps[k], FX::scale(exU, k0 + k));
            }
            put_state(c + 1);
        }
        if (LAG) __syncthreads();   // the side warps' last chunk
        if (d.hT) {
#pragma unroll
            for (int t = 0; t < KTW; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = (w * KTW + t) * 8 + c2 + (e & 1);
                    if (i < d.dk && cok[e >> 1]) d.hT[sbase + (size_t)i * d.dv + col[e >> 1]] = S[t][e];
                }
        }
    } else {
        // side warps: O^T = e^gamma S^T Q^T + U^T P^T, and what the backward reads
        __syncthreads();
        float O[2][4];
        const auto from_state = [&](int c) {   // the first term
            const unsigned char* exS = bufS(c);
            const uint32_t st = front(c);
            const float* tw = factors(slot) + w * 16 + c2;
            const size_t fb = (((size_t)(chunk0 + c) * d.Hv + hv) * d.units + u);
            float part[2][4];
            zero(O);
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const float f = FS::scale(exS, s * KBW);
                zero(part);
#pragma unroll
                for (int b = 0; b < KBW; b++) {
                    const int kk = s * KBW + b;
                    uint32_t a[2][4];
                    FS::template get<2>(exS, kk, lane, a);
                    if (KEEP && on && s == w) put_frag<2, DKP>(d.Sh + fb * 2 * 16 * DKP, 16 * DKP, lane, kk * 16, a);
                    const uint32_t o = wide_off<C>(w * 16 + lb_row(lane), kk * 16 + lb_col(lane));
                    mma_row<2, NPK>(part, a, 0, 1, [&](int p, int, uint32_t (&b4)[4]) { ldm4(b4, st + ST::oQ + p * PK + o); });
                }
                add_scaled(O, part, f);
                if (KEEP && on && s == w && lane == 0) d.mx[(fb * 4 + w) * MX_ROWS + MX_S] = f;
            }
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + (e & 1);
                    O[t][e] *= tw[TOK_EG * C + i] * tw[TOK_FQ * C + i];
                }
        };
        const auto from_chunk = [&](int c, int s) {   // the second (P in stage s), and out
            const uint32_t st = rear(s);
            const float* tk = factors(s);
            const float* tw = tk + w * 16 + c2;
            const size_t fb = (((size_t)(chunk0 + c) * d.Hv + hv) * d.units + u);
            float W[2][4], part[2][4], dn, up;
            get_acc(bufW(c), w * 2, lane, W);
            if (KEEP && on) {
                uint32_t a[2][4];
                frag_scale(W, up, dn);
                frag_pieces<2>(W[0], W[1], up, a);
                put_frag<2, 64>(d.Wh + fb * 2 * 16 * C, 16 * C, lane, w * 16, a);
                put_acc((unsigned char*)(d.Wf + fb * 16 * C), w * 2, lane, W);
                if (lane == 0) d.mx[(fb * 4 + w) * MX_ROWS + MX_W] = dn;
            }
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) W[t][e] *= tw[TOK_BETA * C + t * 8 + (e & 1)];   // U
            frag_scale(W, up, dn);
            FX::put(exO, w, lane, W, up, dn);
            side_bar(grp);
            const float fp = tk[TOK_MISC * C + 4 + w];
#pragma unroll
            for (int kk = 0; kk < C / 16; kk++) {   // row i of P reaches columns j <= i only
                if (kk > w) continue;
                uint32_t a[2][4];
                FX::template get<2>(exO, kk, lane, a);
                const uint32_t o = tile_off<C>(w * 16 + lb_row(lane), kk * 16 + lb_col(lane));
                zero(part);
                mma_row<2, 2>(part, a, 0, 1, [&](int p, int, uint32_t (&f)[4]) { ldm4(f, st + p * ST::TT + o); });
                add_scaled(O, part, FX::scale(exO, kk) * fp);
            }
            const long long t0 = (long long)c * C + w * 16;
            IO* po = (IO*)d.o + (start + t0) * d.ld_o + (long long)hv * d.dv + col[0];
#pragma unroll
            for (int t = 0; t < 2; t++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + c2 + (e & 1);
                    O[t][e] *= d.scale;
                    if (t0 + i < len && cok[e >> 1]) stt(po + (long long)i * ldo, (e >> 1) * 8, O[t][e]);
                }
            }
            if (KEEP && on) put_acc((unsigned char*)(d.Of + fb * 16 * C), w * 2, lane, O);
        };
        for (int c = 0; c < nch; c++) {
            if (!begin(c)) return;
            if (LAG && c > 0) {
                from_chunk(c - 1, last_slot);
            }
            from_state(c);
            if (!LAG) {
                unit_bar(grp);
                from_chunk(c, slot);
            }
        }
        if (LAG) {
            __syncthreads();
            if (nch > 0) from_chunk(nch - 1, slot);
        }
    }
}

template <int DKP, typename IO, bool KEEP, int NU>
cudaError_t go(const DeltaDesc& d, cudaStream_t st) {
    constexpr int SMEM = FwdSmem<DKP, IO>::bytes(NU);
    static_assert(SMEM + NU * 2048 + 128 <= 227 * 1024, "shared memory of a block");
    auto kern = delta_chain_fwd_kernel<DKP, IO, KEEP, NU>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return e;
    const long long blocks = (long long)d.nseq * d.Hv * ((d.units + NU - 1) / NU);
    const int vec = sizeof(IO) == 2 && d.dv % 8 == 0 && d.ld_v % 8 == 0 && ((uintptr_t)d.v & 15) == 0;
    return launch(kern, dim3((unsigned)blocks), dim3(256 * NU), SMEM, st, d.nch > 0, d, vec);
}
template <int DKP, typename IO>
cudaError_t pick(const DeltaDesc& d, bool keep, cudaStream_t st) {
    // two units with fp32 tiles of dk = 128 exceed the shared memory of a block
    if constexpr (!(DKP == 128 && sizeof(IO) == 4)) {
        if (delta_units(d) > 1) return keep ? go<DKP, IO, true, 2>(d, st) : go<DKP, IO, false, 2>(d, st);
    }
    return keep ? go<DKP, IO, true, 1>(d, st) : go<DKP, IO, false, 1>(d, st);
}
}  // namespace

cudaError_t delta_chain_fwd(const DeltaDesc& d, int DKP, bool bf16, bool keep, cudaStream_t st) {
    if (bf16) return DKP == 64 ? pick<64, __nv_bfloat16>(d, keep, st) : pick<128, __nv_bfloat16>(d, keep, st);
    return DKP == 64 ? pick<64, float>(d, keep, st) : pick<128, float>(d, keep, st);
}
}  // namespace kmb
