// delta_bwd.cu -- gated delta rule, backward.
//
// With the chunk's T and P (kmb_delta.cuh) the adjoint is, from the last chunk
// to the first,
//   dU = scale P^T dO + diag(G_C.) K dS_C;   dR = T^T dU;   dV = beta dR
//   dS_0 = e^gamma_C dS_C + scale (e^gamma Q)^T dO - (beta e^gamma K)^T dR
// the forward's three products again, run the other way by the same scheme
// (kmb_delta.cuh).  P^T dO and (e^gamma Q)^T dO carry nothing from chunk to chunk:
// the side warps compute them ahead.  All else has no
// recurrence and is a second kernel, one block per chunk and key head:
//   dP = scale dO U^T (j <= i);   dA = -dR U^T (j < i)
//   dQ = scale e^gamma dO S_0^T + (dP*G) K
//   dK = (beta dA*G) K - beta e^gamma dR S_0^T + (dP*G)^T Q + (beta dA*G)^T K + diag(G_C.) U dS_C^T
// The gradients of the gates need no product over dk.  Scaling a token's decay
// scales o_t against everything it was made of, and summing the adjoints of all
// factors e^gamma leaves
//   dgamma_t = do_t.o_t - v_t.dv_t;   dg_t = <S_0, dS_0> - sum_{s < t in chunk} dgamma_s
// (the state's inner product at the chunk's start anchors the sum, so errors do
// not add up along the sequence), and dbeta_t = dR_t.w_t.  Both are sums
// over dv of what the recurrences leave in fp32.
//
// Measured (8 x 4096 tokens, 8 heads of 64, bf16): recurrence 195 us (3.0 us a
// chunk; bound by the side warps' instructions, then by the chain's latency); dV and
// the gates end some 66 us after it (launched early, so their own time overlaps it); the
// other gradients 231 us (0.30 of the issue slots at 512 chunks and heads, waiting on
// barriers, loads and products in turn).  One
// piece of every factor, 11 bits, took 182 and 183 us, and put the results 1e-3 off
// the fp32 sums rounded to bf16.
#include "kmb_delta.cuh"
#include "kmb_launch.cuh"

namespace kmb {
namespace {

template <int DKP, typename IO>
struct BwdSmem {
    static constexpr int C = kDeltaC, NPK = sizeof(IO) == 4 ? 2 : 1, KT = DKP / 8;
    using ST = DeltaStage<C, DKP, NPK>;
    using FS = FragBuf<DKP / 16, 2>;
    using FX = FragBuf<C / 16, 2>;
    using FG = FragBuf<C / 16, NPK>;
    // of a unit: fragments of dS, dU, of dO and dR with the factors of the state's products; accumulators of the
    // state's product with dO.  dO's fragments share dU's place (the side warps use it after a chunk's dU is read),
    // P^T dO, from the side warps for the next chunk, shares that of dR, to them.
    static constexpr int oX = FS::BYTES, oE = oX + FX::BYTES, oF = oE + FX::BYTES, oR = oF + FX::BYTES, oZ = oR + 4096,
                         EX = oZ + KT * 512;
    static constexpr int bytes(int nu) { return 2 * ST::BYTES + nu * EX; }
};

template <int DKP, typename IO, int NU>
__global__ void __launch_bounds__(256 * NU, 1)
delta_chain_bwd_kernel(const __grid_constant__ DeltaDesc d, int vec) {
    using SM = BwdSmem<DKP, IO>;
    constexpr int C = kDeltaC, NPK = SM::NPK;
    using ST = typename SM::ST;
    using FS = typename SM::FS;
    using FX = typename SM::FX;
    using FG = typename SM::FG;
    constexpr int KT = DKP / 8, KTW = KT / 4, KBW = DKP / 64;
    constexpr int PK = C * DKP * 2;
    extern __shared__ __align__(128) unsigned char sm[];
    constexpr int NS = 2;   // stages of tiles (a third changed nothing: 204 us against 203)
    __shared__ __align__(8) uint64_t full[NS];
    const uint32_t sb = (uint32_t)__cvta_generic_to_shared(sm);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = warp >> 3, w = warp & 3;
    const bool chain = (warp & 4) == 0;
    unsigned char* exS = sm + NS * ST::BYTES + grp * SM::EX;
    unsigned char *exX = exS + SM::oX, *exE = exS + SM::oE, *exF = exS + SM::oF, *exR = exS + SM::oR, *exZ = exS + SM::oZ;
    const int ub = (d.units + NU - 1) / NU;
    const int u = (int)(blockIdx.x % ub) * NU + grp;
    const int hv = (int)(blockIdx.x / ub) % d.Hv, nr = (int)(blockIdx.x / ub) / d.Hv;
    pdl_release();
    const int n = d.order ? d.order[nr] : nr;
    const bool on = u < d.units;
    const int r = lane >> 2, c2 = (lane & 3) * 2;
    const int col[2] = {u * 16 + r, u * 16 + r + 8};
    const bool cok[2] = {col[0] < d.dv, col[1] < d.dv};
    long long start, len;
    seq_range(d, n, start, len);
    const int chunk0 = d.cu ? d.cstart[n] : n * d.nc;
    const int nch = (int)((len + C - 1) / C);
    const size_t sbase = ((size_t)n * d.Hv + hv) * d.dk * d.dv;

    const auto stage = [&](int i) { return i % NS; };
    // the chain warps of the first unit copy the tiles of the recurrence's step i (the side warps have more to do)
    const bool copies = warp < 4 && lane == 0;
    const auto fetch = [&](int i) {
        const uint32_t st = sb + stage(i) * ST::BYTES;
        ST::load(d, d.Tt, st, st + ST::FRONT, smem_u32(&full[stage(i)]), chunk0 + nch - 1 - i, hv, w);
    };
    const auto arrived = [&](int i) { return mbar_wait(smem_u32(&full[stage(i)]), (i / NS) & 1); };
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; i++) mbar_init(smem_u32(&full[i]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (copies)
        for (int i = 0; i < NS - 1 && i < nch; i++) fetch(i);
    // The chunk's tiles are there, the state's fragments too, and the last chunk's stage is read; false: a wait ran out.
    const auto begin = [&](int i) {
        const bool got = arrived(i);
        if (!__syncthreads_and(got)) {
            if (!got) {
                set_status(d.status, KMB_ERR_TIMEOUT_FULL);
                arrived(i);   // the block's memory stays its own for another limit
            }
            return false;
        }
        if (copies && i + NS - 1 < nch) fetch(i + NS - 1);
        return true;
    };

    if (chain) {
        float S[KTW][4], up, dn;   // dS^T, the warp's quarter of dk
#pragma unroll
        for (int t = 0; t < KTW; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = (w * KTW + t) * 8 + c2 + (e & 1);
                S[t][e] = (d.dhT && i < d.dk && cok[e >> 1]) ? d.dhT[sbase + (size_t)i * d.dv + col[e >> 1]] : 0.0f;
            }
        const auto put_state = [&]() {
            frag_scale(S, up, dn);
#pragma unroll
            for (int b = 0; b < KBW; b++) {
                uint32_t a[2][4];
                frag_pieces<2>(S[2 * b], S[2 * b + 1], up, a);
                FS::put(exS, w * KBW + b, lane, a, dn);
            }
        };
        put_state();
        __syncthreads();
        for (int it = 0; it < nch; it++) {
            if (!begin(it)) return;
            const uint32_t st = sb + stage(it) * ST::BYTES;
            const float* tk = (const float*)(sm + stage(it) * ST::BYTES + ST::FRONT + ST::oTok);
            const float* tw = tk + w * 16 + c2;
            // dU = diag(G_C.) K dS_C + scale P^T dO (the latter from the side warps)
            float X[2][4], Y[2][4], part[2][4];
            zero(X);
#pragma unroll
            for (int s = 0; s < 4; s++) {
                zero(part);
#pragma unroll
                for (int b = 0; b < KBW; b++) {
                    const int kk = s * KBW + b;
                    uint32_t a[2][4];
                    FS::template get<2>(exS, kk, lane, a);
                    const uint32_t o = wide_off<C>(w * 16 + lb_row(lane), kk * 16 + lb_col(lane));
                    mma_row<2, NPK>(part, a, 0, 1, [&](int p, int, uint32_t (&f)[4]) { ldm4(f, st + p * PK + o); });
                }
                add_scaled(X, part, FS::scale(exS, s * KBW));
            }
            get_acc(exR, w * 2, lane, Y);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + (e & 1);
                    X[t][e] = fmaf(X[t][e], tw[TOK_GC * C + i] * tw[TOK_FK * C + i], Y[t][e]);
                    Y[t][e] = 0.0f;
                }
            frag_scale(X, up, dn);
            FX::put(exX, w, lane, X, up, dn);
            chain_bar(grp);
            // dR^T = dU^T T: column j of T has rows i >= j only
#pragma unroll
            for (int kk = 0; kk < C / 16; kk++) {
                if (kk < w) continue;
                uint32_t a[2][4];
                FX::template get<2>(exX, kk, lane, a);
                const uint32_t o = tile_off<C>(kk * 16 + la_row(lane), w * 16 + la_col(lane));
                zero(part);
                mma_row<2, 2>(part, a, 0, 1, [&](int p, int, uint32_t (&f)[4]) { ldm4t(f, st + ST::oT + p * ST::TT + o); });
                add_scaled(Y, part, FX::scale(exX, kk) * tk[TOK_MISC * C + 8 + kk]);
            }
            put_acc(exR, w * 2, lane, Y);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + (e & 1);
                    X[t][e] = Y[t][e] * -(tw[TOK_BETA * C + i] * tw[TOK_EG * C + i] * tw[TOK_FK * C + i]);
                }
            frag_scale(X, up, dn);
            FX::put(exF, w, lane, X, up, dn);
            unit_bar(grp);
            // dS^T <- e^gamma_C dS^T + (scale e^gamma dO)^T Q (from the side warps) - (beta e^gamma dR)^T K
            const float last = tk[TOK_EG * C + C - 1];
            float ps[KTW][4];
            get_acc(exZ, w * KTW, lane, ps);
#pragma unroll
            for (int t = 0; t < KTW; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) S[t][e] = fmaf(S[t][e], last, ps[t][e]);
#pragma unroll
            for (int kk = 0; kk < C / 16; kk++) {
                uint32_t a[2][4];
                FX::template get<2>(exF, kk, lane, a);
                zero(ps);
                mma_row<2, NPK>(ps, a, 0, KTW / 2, [&](int p, int t2, uint32_t (&f)[4]) {
                    ldm4t(f, st + p * PK + wide_off<C>(kk * 16 + la_row(lane), (w * KTW + t2 * 2) * 8 + la_col(lane)));
                });
                add_scaled(S, ps, FX::scale(exF, kk));
            }
            put_state();
        }
        __syncthreads();   // the side warps read the last fragments
        if (d.dh0) {
#pragma unroll
            for (int t = 0; t < KTW; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = (w * KTW + t) * 8 + c2 + (e & 1);
                    if (i < d.dk && cok[e >> 1]) d.dh0[sbase + (size_t)i * d.dv + col[e >> 1]] = S[t][e];
                }
        }
        return;
    }

    // side warps
    TokenTile<IO> Gn;
    const auto load_go = [&](int c) {
        const long long t0 = (long long)c * C + w * 16;
        Gn.load(d.go, start + t0, d.ld_do, (long long)hv * d.dv + u * 16, on ? d.dv - u * 16 : 0,
                (int)(len - t0 < 16 ? len - t0 : 16), lane, vec);
    };
    const auto unit_at = [&](int c) { return ((size_t)(chunk0 + c) * d.Hv + hv) * d.units + u; };
    float G[2][4], part[2][4], up, dn;   // dO^T of the warp's tokens
    // ahead of chunk c (tile stage `s`): dO's fragments, plain and with the factors of the state's product; P^T dO
    const auto ahead = [&](int c, int s) {
        const uint32_t st = sb + s * ST::BYTES;
        const float* tk = (const float*)(sm + s * ST::BYTES + ST::FRONT + ST::oTok);
        const float* tw = tk + w * 16 + c2;
        uint32_t a[NPK][4];
        Gn.tiles(G, exR + w * 1024, lane, vec);   // the place of the dR that this warp has read
        frag_scale(G, up, dn);
        frag_pieces<NPK>(G[0], G[1], up, a);
        FG::put(exX, w, lane, a, dn);
        if (on) {
            const size_t fb = unit_at(c);
            put_frag<NPK, 64>(d.Gh + fb * NPK * 16 * C, 16 * C, lane, w * 16, a);
            if (lane == 0) d.mx[(fb * 4 + w) * MX_ROWS + MX_DO] = dn;
        }
        float Y[2][4];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = t * 8 + (e & 1);
                Y[t][e] = G[t][e] * (d.scale * tw[TOK_EG * C + i] * tw[TOK_FQ * C + i]);
            }
        frag_scale(Y, up, dn);
        FX::put(exE, w, lane, Y, up, dn);
        side_bar(grp);
        zero(Y);
#pragma unroll
        for (int kk = 0; kk < C / 16; kk++) {   // column j of P has rows i >= j only
            if (kk < w) continue;
            uint32_t a1[NPK][4];
            FG::template get<NPK>(exX, kk, lane, a1);
            const uint32_t o = tile_off<C>(kk * 16 + la_row(lane), w * 16 + la_col(lane));
            zero(part);
            mma_row<NPK, 2>(part, a1, 0, 1, [&](int p, int, uint32_t (&f)[4]) { ldm4t(f, st + ST::FRONT + p * ST::TT + o); });
            add_scaled(Y, part, FG::scale(exX, kk) * (tk[TOK_MISC * C + 4 + kk] * d.scale));
        }
        put_acc(exR, w * 2, lane, Y);
    };
    float sr[KTW][4];   // the warp's part of the state at the start of the last chunk done
    zero(sr);
    // <S_0, dS_0> at the start of chunk c, from the fragments that the chain left
    const auto anchor = [&](int c) {
        float an = 0.0f;
#pragma unroll
        for (int b = 0; b < KBW; b++) {
            uint32_t a[2][4];
            FS::template get<2>(exS, w * KBW + b, lane, a);
#pragma unroll
            for (int i = 0; i < 4; i++) {   // fragment word i: row half i & 1, tile i >> 1
                const float2 x = join(a[0][i], a[1][i]);
                const float (&y)[4] = sr[2 * b + (i >> 1)];
                an = fmaf(x.x, y[(i & 1) * 2], an);
                an = fmaf(x.y, y[(i & 1) * 2 + 1], an);
            }
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) an += __shfl_xor_sync(0xffffffffu, an, o);
        if (on && lane == 0) d.anchor[unit_at(c) * 4 + w] = an * FS::scale(exS, w * KBW);
    };
    if (nch > 0) load_go(nch - 1);
    __syncthreads();
    if (nch > 0) {
        if (!arrived(0)) set_status(d.status, KMB_ERR_TIMEOUT_FULL);
        ahead(nch - 1, 0);
    }
    for (int it = 0; it < nch; it++) {
        const int c = nch - 1 - it;
        if (!begin(it)) return;
        const uint32_t st = sb + stage(it) * ST::BYTES;
        const size_t fb = unit_at(c);
        float* mx = d.mx + (fb * 4 + w) * MX_ROWS;
        if (c > 0) load_go(c - 1);   // in flight under the products
        // keep dS_C; its product with the state at the same place
        if (it > 0) anchor(c + 1);
#pragma unroll
        for (int b = 0; b < KBW; b++) {
            uint32_t a[2][4];
            FS::template get<2>(exS, w * KBW + b, lane, a);
            if (on) {
                put_frag<2, DKP>(d.dSh + fb * 2 * 16 * DKP, 16 * DKP, lane, (w * KBW + b) * 16, a);
                if (lane == 0) mx[MX_DS] = FS::scale(exS, w * KBW);
            }
        }
        if (on) get_acc((const unsigned char*)(d.Sf + fb * 16 * DKP), w * KTW, lane, sr);
        // (scale e^gamma dO)^T Q
        {
            float Z[KTW][4], ps[KTW][4];
            zero(Z);
#pragma unroll
            for (int kk = 0; kk < C / 16; kk++) {
                uint32_t a[2][4];
                FX::template get<2>(exE, kk, lane, a);
                zero(ps);
                mma_row<2, NPK>(ps, a, 0, KTW / 2, [&](int p, int t2, uint32_t (&f)[4]) {
                    ldm4t(f, st + ST::oQ + p * PK +
                                 wide_off<C>(kk * 16 + la_row(lane), (w * KTW + t2 * 2) * 8 + la_col(lane)));
                });
                add_scaled(Z, ps, FX::scale(exE, kk));
            }
            put_acc(exZ, w * KTW, lane, Z);
        }
        unit_bar(grp);
        float Y[2][4];   // dR, kept
        get_acc(exR, w * 2, lane, Y);
        if (on) {
            uint32_t a[2][4];
            frag_scale(Y, up, dn);
            frag_pieces<2>(Y[0], Y[1], up, a);
            put_frag<2, 64>(d.Rh + fb * 2 * 16 * C, 16 * C, lane, w * 16, a);
            if (lane == 0) mx[MX_R] = dn;
            put_acc((unsigned char*)(d.Rf + fb * 16 * C), w * 2, lane, Y);
        }
        if (c > 0) {
            if (!arrived(it + 1)) set_status(d.status, KMB_ERR_TIMEOUT_FULL);
            ahead(c - 1, stage(it + 1));
        }
    }
    __syncthreads();
    if (nch > 0) anchor(0);
}

// ------------------------------------------------------------------ dV and the gates
// Block = (chunk, value head), warp = 16 of its tokens over all of dv: dV = beta dR, and per token the sums over dv
// that the gates' gradients are made of.  Bound by what it reads and writes: 5 dv + 3 dv bytes in fp32 and bf16 a
// token, in accumulator order so that every load but v's is a whole line.
template <typename IO>
__global__ void __launch_bounds__(128)
delta_gates_kernel(const __grid_constant__ DeltaDesc d) {
    constexpr int C = kDeltaC, NP = sizeof(IO) == 4 ? 2 : 1;
    using RT = typename RawOf<IO>::type;
    __shared__ float sums[2][C];
    const int lane = threadIdx.x & 31, wb = threadIdx.x >> 5;
    const int r = lane >> 2, c2 = (lane & 3) * 2;
    const int chunk = blockIdx.x, hv = blockIdx.y;
    long long tok0;
    int cnt;
    pdl_release();
    if (!chunk_range<C>(d, chunk, tok0, cnt)) return;   // the offsets are the forward's
    pdl_wait();
    const size_t head = (size_t)chunk * d.Hv + hv;
    const int ldv = (int)d.ld_v, lddv = (int)d.ld_dv;
    const float* tk = d.tok + head * TOK_SIZE + TOK_BETA * C + wb * 16 + c2;
    const float2 be[2] = {*(const float2*)tk, *(const float2*)(tk + 8)};
    float ts[2][2] = {}, bs[2][2] = {};
#pragma unroll 2
    for (int u = 0; u < d.units; u++) {
        const size_t fb = head * d.units + u;
        const float* mx = d.mx + (fb * 4 + wb) * MX_ROWS;
        const int c0 = u * 16 + r;
        const bool ok[2] = {c0 < d.dv, c0 + 8 < d.dv};
        const RT* pv = (const RT*)d.v + (tok0 + wb * 16) * d.ld_v + (long long)hv * d.dv + c0;
        IO* pd = (IO*)d.dvv + (tok0 + wb * 16) * d.ld_dv + (long long)hv * d.dv + c0;
        float O[2][4], R[2][4], W[2][4];
        uint32_t G[2][2][2];
        RT V[2][4];
        get_acc((const unsigned char*)(d.Of + fb * 16 * C), wb * 2, lane, O);
        get_acc((const unsigned char*)(d.Rf + fb * 16 * C), wb * 2, lane, R);
        get_acc((const unsigned char*)(d.Wf + fb * 16 * C), wb * 2, lane, W);
#pragma unroll
        for (int t = 0; t < 2; t++) {
            get_tile<64, NP>(d.Gh + fb * NP * 16 * C, 16 * C, lane, wb * 16 + t * 8, G[t]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = t * 8 + c2 + (e & 1);
                V[t][e] = (wb * 16 + i < cnt && ok[e >> 1]) ? pv[(long long)i * ldv + (e >> 1) * 8] : RT(0);
            }
        }
        const float sG = mx[MX_DO];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float2 g2 = NP == 2 ? join(G[t][h][0], G[t][h][1])
                                          : __half22float2(*reinterpret_cast<const __half2*>(&G[t][h][0]));
                const float gg[2] = {g2.x * sG, g2.y * sG};
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int i = t * 8 + c2 + e;
                    const float dv = (e ? be[t].y : be[t].x) * R[t][h * 2 + e];
                    bs[t][e] = fmaf(R[t][h * 2 + e], W[t][h * 2 + e], bs[t][e]);
                    ts[t][e] = fmaf(gg[e], O[t][h * 2 + e], ts[t][e]);
                    ts[t][e] = fmaf(-from_raw(V[t][h * 2 + e]), dv, ts[t][e]);
                    if (wb * 16 + i < cnt && ok[h]) stt(pd + (long long)i * lddv, h * 8, dv);
                }
            }
    }
    if (!d.dg && !d.dbeta) return;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                ts[t][e] += __shfl_xor_sync(0xffffffffu, ts[t][e], o);
                bs[t][e] += __shfl_xor_sync(0xffffffffu, bs[t][e], o);
            }
    if (r < 2) {   // row r of the lanes writes tile r
        sums[0][wb * 16 + r * 8 + c2] = r ? ts[1][0] : ts[0][0];
        sums[0][wb * 16 + r * 8 + c2 + 1] = r ? ts[1][1] : ts[0][1];
        sums[1][wb * 16 + r * 8 + c2] = r ? bs[1][0] : bs[0][0];
        sums[1][wb * 16 + r * 8 + c2 + 1] = r ? bs[1][1] : bs[0][1];
    }
    __syncthreads();
    if (wb) return;
    // one warp: running sums over the chunk's tokens (lane and lane + 32) from <S_0, dS_0>
    double anchor = lane < d.units * 4 ? (double)d.anchor[head * d.units * 4 + lane] : 0.0;
    const double t[2] = {sums[0][lane], sums[0][lane + 32]};
    double s[2] = {t[0], t[1]};
#pragma unroll
    for (int o = 16; o; o >>= 1) anchor += __shfl_xor_sync(0xffffffffu, anchor, o);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, s[0], o), y = __shfl_up_sync(0xffffffffu, s[1], o);
        if (lane >= o) {
            s[0] += x;
            s[1] += y;
        }
    }
    s[1] += __shfl_sync(0xffffffffu, s[0], 31);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int i = h * 32 + lane;
        if (i >= cnt) continue;
        const long long at = (tok0 + i) * d.Hv + hv;
        // a decay below e^-104 is 0 in fp32: nothing depends on it
        const bool reset = d.g && d.g[at] < -104.0f;
        if (d.dg) d.dg[at] = reset ? 0.0f : (float)(anchor - (s[h] - t[h]));
        if (d.dbeta) d.dbeta[at] = sums[1][i];
    }
}

// ------------------------------------------------------------------ gradients without recurrence
// Eight warps: 16 token rows x half of dk (and half of the 64 columns of dP, dA) each.  dv is walked in slices of
// four units, whose fp16 tiles come as the recurrences left them: one piece for what is exact in one (K, Q and dO in
// bf16), two for all else, so that dQ and dK are fp32 sums rounded once.  A unit is one step of 16 in the products over dv, so its powers of two are
// applied when the step's products are added to the fp32 sums.
template <int DKP, int NK>
struct GradSmem {
    static constexpr int C = kDeltaC, NH = DKP / 64;
    static constexpr int KQ = NK * C * DKP * 2, T64 = 64 * C * 2, SD = NH * 64 * 128;
    static constexpr int oK = 0, oQ = KQ, oG = 2 * KQ, oW = oG + NK * T64, oR = oW + 2 * T64, oS = oR + 2 * T64,
                         oD = oS + 2 * SD, oEnd = oD + 2 * SD;
    // the four weighted matrices take the place of the slices
    static constexpr int oE = oG, TE = C * C * 2;
    static constexpr int oTok = (oE + 8 * TE > oEnd ? oE + 8 * TE : oEnd);
    static constexpr int oMx = oTok + TOK_SIZE * 4;
    static constexpr int oGam = oMx + 8 * 4 * MX_ROWS * 4;
    static constexpr int oRow = oGam + C * 8, oCol = oRow + C * 4;
    static constexpr int BYTES = oCol + 3 * 48 * 4;
};

template <int DKP, typename IO>
__global__ void __launch_bounds__(256, DKP == 64 ? 2 : 1)
delta_grads_kernel(const __grid_constant__ DeltaDesc d) {
    constexpr int C = kDeltaC;
    constexpr int NK = sizeof(IO) == 4 ? 2 : 1;   // pieces of K, Q and dO
    using SM = GradSmem<DKP, NK>;
    constexpr int HN = DKP / 2, HT = HN / 8;
    constexpr int PK = C * DKP * 2;
    extern __shared__ __align__(128) unsigned char sm[];
    __shared__ float wf[4][4][4];   // of the weighted matrices: what block (row block, column block) is times
    const uint32_t sb = (uint32_t)__cvta_generic_to_shared(sm);
    float* tk = (float*)(sm + SM::oTok);
    float* mx = (float*)(sm + SM::oMx);
    DecaySmem dec{(double*)(sm + SM::oGam), (float*)(sm + SM::oRow), (float*)(sm + SM::oCol)};
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rg = warp & 3, ch = warp >> 2;
    const int r = lane >> 2, c2 = (lane & 3) * 2;
    const int chunk = blockIdx.x, hk = blockIdx.y;
    long long tok0;
    int cnt;
    if (!chunk_range<C>(d, chunk, tok0, cnt)) return;   // the offsets are the forward's
    {
        const char* ks = (const char*)(d.Kt + ((size_t)chunk * d.Hk + hk) * NK * C * DKP);
        const char* qs = (const char*)(d.Qt + ((size_t)chunk * d.Hk + hk) * NK * C * DKP);
        for (int i = tid; i < SM::KQ / 16; i += 256) {
            cp16(sb + SM::oK + i * 16, ks + i * 16);
            cp16(sb + SM::oQ + i * 16, qs + i * 16);
        }
        cp_commit();
    }
    pdl_wait();
    float dQ[HT][4], dK[HT][4];
    zero(dQ);
    zero(dK);

    for (int hh = 0; hh < d.grp; hh++) {
        const int hv = hk * d.grp + hh;
        const size_t head = (size_t)chunk * d.Hv + hv;
        // tiles of units u0 .. u0 + 3
        const auto slice = [&](int u0) {
            const int nx = d.units - u0 < 4 ? d.units - u0 : 4;
            for (int i = tid; i < nx * 256; i += 256) {
                const int x = i / 256, p = i / 128 % 2, o = (i & 127) * 16;
                const size_t un = head * d.units + u0 + x, g = (un * 2 + p) * 2048 + o;
                const uint32_t s = sb + p * SM::T64 + x * 2048 + o;
                if (p < NK) cp16(s + SM::oG, (const char*)d.Gh + (un * NK + p) * 2048 + o);
                cp16(s + SM::oR, (const char*)d.Rh + g);
                cp16(s + SM::oW, (const char*)d.Wh + g);
            }
            for (int i = tid; i < nx * 2 * SM::NH * 128; i += 256) {
                const int x = i / (2 * SM::NH * 128), p = i / (SM::NH * 128) % 2, h = i / 128 % SM::NH, o = (i & 127) * 16;
                const size_t g = (((head * d.units + u0 + x) * 2 + p) * SM::NH + h) * 2048 + o;
                const uint32_t s = sb + p * SM::SD + h * 8192 + x * 2048 + o;
                cp16(s + SM::oD, (const char*)d.dSh + g);
                cp16(s + SM::oS, (const char*)d.Sh + g);
            }
            cp_commit();
        };
        __syncthreads();
        for (int i = tid; i < TOK_SIZE / 4; i += 256) cp16(sb + SM::oTok + i * 16, d.tok + head * TOK_SIZE + i * 4);
        for (int i = tid; i < d.units * MX_ROWS; i += 256) cp16(sb + SM::oMx + i * 16, d.mx + head * d.units * 4 * MX_ROWS + i * 4);
        for (int i = tid; i < C / 2; i += 256) cp16(sb + SM::oGam + i * 16, d.gam + head * C + i * 2);
        slice(0);
        cp_wait<0>();
        __syncthreads();
        decay_tables(dec, tid);

        float dP[4][4], dA[4][4];
        zero(dP);
        zero(dA);
        float fq[2], fz[2], fu[2];   // row factors of the products with the states
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int i = rg * 16 + r + h * 8;
            const float eg = tk[TOK_EG * C + i], be = tk[TOK_BETA * C + i];
            fq[h] = d.scale * eg;
            fz[h] = -be * eg;
            fu[h] = tk[TOK_GC * C + i] * be;
        }
        for (int u0 = 0; u0 < d.units; u0 += 4) {
            if (u0) {
                __syncthreads();
                slice(u0);
                cp_wait<0>();
                __syncthreads();
            }
            const int nx = d.units - u0 < 4 ? d.units - u0 : 4;
            for (int kk = 0; kk < nx; kk++) {
                const float* m4 = mx + (u0 + kk) * 4 * MX_ROWS;
                const float sG = m4[rg * MX_ROWS + MX_DO], sR = m4[rg * MX_ROWS + MX_R], sW = m4[rg * MX_ROWS + MX_W];
                uint32_t aG[NK][4], aR[2][4], aW[2][4];
                const uint32_t oa = tile_off<64>(kk * 16 + lb_row(lane), rg * 16 + lb_col(lane));
#pragma unroll
                for (int p = 0; p < NK; p++) ldm4t(aG[p], sb + SM::oG + p * SM::T64 + oa);
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    ldm4t(aR[p], sb + SM::oR + p * SM::T64 + oa);
                    ldm4t(aW[p], sb + SM::oW + p * SM::T64 + oa);
                }
                // dO W^T and dR W^T, columns up to the diagonal block
#pragma unroll
                for (int t2 = 0; t2 < 2; t2++) {
                    if (ch * 2 + t2 > rg) continue;
                    const float sw = m4[(ch * 2 + t2) * MX_ROWS + MX_W];
                    const auto ldw = [&](int p, int, uint32_t (&b)[4]) {
                        ldm4t(b, sb + SM::oW + p * SM::T64 + tile_off<64>(kk * 16 + la_row(lane), ch * 32 + t2 * 16 + la_col(lane)));
                    };
                    float part[2][4], par2[2][4];
                    zero(part);
                    zero(par2);
                    mma_row<NK, 2>(part, aG, 0, 1, ldw);
                    mma_row<2, 2>(par2, aR, 0, 1, ldw);
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            dP[t2 * 2 + t][e] = fmaf(part[t][e], sG * sw, dP[t2 * 2 + t][e]);
                            dA[t2 * 2 + t][e] = fmaf(par2[t][e], sR * sw, dA[t2 * 2 + t][e]);
                        }
                }
                // dO S_0^T, dR S_0^T, W dS_C^T: columns in quarters of dk, two of them this warp's
#pragma unroll
                for (int qd = 0; qd < 2; qd++) {
                    constexpr int QT = DKP / 32;   // tiles of a quarter
                    const float* mq = m4 + (ch * 2 + qd) * MX_ROWS;
                    const float sS = mq[MX_S], sD = mq[MX_DS];
                    float part[QT][4];
                    const auto ld_at = [&](int base, int p, int t2, uint32_t (&b)[4]) {
                        ldm4t(b, sb + base + p * SM::SD +
                                     wide_off<64>(kk * 16 + la_row(lane), ch * HN + qd * QT * 8 + t2 * 16 + la_col(lane)));
                    };
                    const auto lds = [&](int p, int t2, uint32_t (&b)[4]) { ld_at(SM::oS, p, t2, b); };
                    const auto ldd = [&](int p, int t2, uint32_t (&b)[4]) { ld_at(SM::oD, p, t2, b); };
                    const auto add = [&](float (&to)[HT][4], const float (&f)[2], float s) {
#pragma unroll
                        for (int t = 0; t < QT; t++)
#pragma unroll
                            for (int e = 0; e < 4; e++) to[qd * QT + t][e] = fmaf(part[t][e], f[e >> 1] * s, to[qd * QT + t][e]);
                    };
                    zero(part);
                    mma_row<NK, 2>(part, aG, 0, QT / 2, lds);
                    add(dQ, fq, sG * sS);
                    zero(part);
                    mma_row<2, 2>(part, aR, 0, QT / 2, lds);
                    add(dK, fz, sR * sS);
                    zero(part);
                    mma_row<2, 2>(part, aW, 0, QT / 2, ldd);
                    add(dK, fu, sW * sD);
                }
            }
        }
        __syncthreads();   // the decay tables are there (with dv <= 64 no slice's barrier came in between)
        // weighted matrices: E = scale G dO U^T with the key's and with the query's tile scale, F = -beta G dR U^T
        // with the key's of either side.  Each block of 16 x 16 has its power of two, like all other factors.
        float eu[4][2];
#pragma unroll
        for (int t2 = 0; t2 < 2; t2++) {
            const int cb = ch * 2 + t2;
            if (cb > rg) continue;
            float m[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int t = t2 * 2; t < t2 * 2 + 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = rg * 16 + r + (e >> 1) * 8, j = ch * 32 + t * 8 + c2 + (e & 1);
                    const float g = dec.at(i, j, cb == rg, rg) * tk[TOK_BETA * C + j];
                    dP[t][e] = j <= i ? g * d.scale * dP[t][e] : 0.0f;
                    dA[t][e] = j < i ? -g * tk[TOK_BETA * C + i] * dA[t][e] : 0.0f;
                    m[0] = fmaxf(m[0], fabsf(dP[t][e] * tk[TOK_FK * C + j]));
                    m[1] = fmaxf(m[1], fabsf(dP[t][e] * tk[TOK_FQ * C + i]));
                    m[2] = fmaxf(m[2], fabsf(dA[t][e] * tk[TOK_FK * C + j]));
                    m[3] = fmaxf(m[3], fabsf(dA[t][e] * tk[TOK_FK * C + i]));
                }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float down;
                warp_scale(m[k], eu[k][t2], down);
                if (lane == 0) wf[k][rg][cb] = down;
            }
        }
        __syncthreads();   // the slices are read
#pragma unroll
        for (int t = 0; t < 4; t++) {
            if (ch * 2 + (t >> 1) > rg) continue;   // blocks above the diagonal are never read
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int i = rg * 16 + r + h * 8, j = ch * 32 + t * 8 + c2;
                const float fki = tk[TOK_FK * C + i], fqi = tk[TOK_FQ * C + i];
                const float f0 = tk[TOK_FK * C + j], f1 = tk[TOK_FK * C + j + 1];
                const float p0 = dP[t][h * 2], p1 = dP[t][h * 2 + 1], a0 = dA[t][h * 2], a1 = dA[t][h * 2 + 1];
                const float v[4][2] = {{p0 * f0, p1 * f1}, {p0 * fqi, p1 * fqi}, {a0 * f0, a1 * f1}, {a0 * fki, a1 * fki}};
                const uint32_t o = tile_off<C>(i, j);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t p[2];
                    split_pair<2>(v[k][0] * eu[k][t >> 1], v[k][1] * eu[k][t >> 1], p);
#pragma unroll
                    for (int x = 0; x < 2; x++) *(uint32_t*)(sm + SM::oE + (k * 2 + x) * SM::TE + o) = p[x];
                }
            }
        }
        __syncthreads();
        // the four products over tokens
#pragma unroll
        for (int k = 0; k < 4; k++) {
            // k: 0 E K -> dQ, 2 F K -> dK (rows i, sum over j <= i); 1 E^T Q, 3 F^T K -> dK (rows j, sum over i >= j)
            float (&to)[HT][4] = k == 0 ? dQ : dK;
#pragma unroll
            for (int kk = 0; kk < C / 16; kk++) {
                if ((k & 1) ? kk < rg : kk > rg) continue;
                uint32_t a[2][4];
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    const uint32_t base = sb + SM::oE + (k * 2 + p) * SM::TE;
                    if (k & 1) ldm4t(a[p], base + tile_off<C>(kk * 16 + lb_row(lane), rg * 16 + lb_col(lane)));
                    else ldm4(a[p], base + tile_off<C>(rg * 16 + la_row(lane), kk * 16 + la_col(lane)));
                }
                float acc[HT][4];
                zero(acc);
                mma_row<2, NK>(acc, a, 0, HN / 16, [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4t(b, sb + (k == 1 ? SM::oQ : SM::oK) + p * PK +
                                 wide_off<C>(kk * 16 + la_row(lane), ch * HN + t2 * 16 + la_col(lane)));
                });
                add_scaled(to, acc, (k & 1) ? wf[k][kk][rg] : wf[k][rg][kk]);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int i = rg * 16 + r + h * 8;
        if (i >= cnt) continue;
        IO* pq = (IO*)d.dq + (tok0 + i) * d.ld_dq + (long long)hk * d.dk;
        IO* pk = (IO*)d.dkk + (tok0 + i) * d.ld_dk + (long long)hk * d.dk;
#pragma unroll
        for (int t = 0; t < HT; t++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int cc = ch * HN + t * 8 + c2 + e;
                if (cc < d.dk) {
                    stt(pq, cc, dQ[t][h * 2 + e]);
                    stt(pk, cc, dK[t][h * 2 + e]);
                }
            }
    }
}

template <int DKP, typename IO, int NU>
cudaError_t chain_go(const DeltaDesc& d, cudaStream_t st) {
    constexpr int SMEM = BwdSmem<DKP, IO>::bytes(NU);
    static_assert(BwdSmem<DKP, IO>::bytes(1) + 64 <= 227 * 1024, "shared memory of a block");
    auto kern = delta_chain_bwd_kernel<DKP, IO, NU>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return e;
    const long long blocks = (long long)d.nseq * d.Hv * ((d.units + NU - 1) / NU);
    const int vec = sizeof(IO) == 2 && d.dv % 8 == 0 && d.ld_do % 8 == 0 && ((uintptr_t)d.go & 15) == 0;
    kern<<<(unsigned)blocks, 256 * NU, SMEM, st>>>(d, vec);
    return cudaGetLastError();
}
template <int DKP, typename IO>
cudaError_t chain_pick(const DeltaDesc& d, cudaStream_t st) {
    if constexpr (!(DKP == 128 && sizeof(IO) == 4)) {
        if (delta_units(d) > 1) return chain_go<DKP, IO, 2>(d, st);
    }
    return chain_go<DKP, IO, 1>(d, st);
}
template <int DKP, typename IO>
cudaError_t grads_go(const DeltaDesc& d, cudaStream_t st) {
    using SM = GradSmem<DKP, sizeof(IO) == 4 ? 2 : 1>;
    auto kern = delta_grads_kernel<DKP, IO>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::BYTES);
    if (e != cudaSuccess) return e;
    e = launch(delta_gates_kernel<IO>, dim3((unsigned)d.nch, (unsigned)d.Hv), dim3(128), 0, st, true, d);
    if (e != cudaSuccess) return e;
    return launch(kern, dim3((unsigned)d.nch, (unsigned)d.Hk), dim3(256), SM::BYTES, st, true, d);
}
}  // namespace

cudaError_t delta_chain_bwd(const DeltaDesc& d, int DKP, bool bf16, cudaStream_t st) {
    if (bf16) return DKP == 64 ? chain_pick<64, __nv_bfloat16>(d, st) : chain_pick<128, __nv_bfloat16>(d, st);
    return DKP == 64 ? chain_pick<64, float>(d, st) : chain_pick<128, float>(d, st);
}
cudaError_t delta_grads(const DeltaDesc& d, int DKP, bool bf16, cudaStream_t st) {
    if (bf16) return DKP == 64 ? grads_go<64, __nv_bfloat16>(d, st) : grads_go<128, __nv_bfloat16>(d, st);
    return DKP == 64 ? grads_go<64, float>(d, st) : grads_go<128, float>(d, st);
}
}  // namespace kmb
