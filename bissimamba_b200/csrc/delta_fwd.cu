// delta_fwd.cu -- gated delta rule, forward recurrence over chunks.
//
// The columns of the state evolve independently, so a warp owns 16 of them and
// keeps the transposed state S^T [16 columns of dv][dk] in registers as
// accumulators of m16n8 products.  Transposed, every product of a chunk takes
// its fp32 factor from the registers of the same warp (an accumulator tile is
// laid out as an A operand) and its other factor from shared memory:
//   (K S)^T = S^T K^T;  W^T = (V - e^gamma K S)^T M^T;  U = beta W;  O^T = e^gamma S^T Q^T + U^T P^T
//   S^T <- e^gamma_C S^T + (G_C. U)^T K
// so the chain of a chunk needs no exchange between warps; the block's warps
// only share the staged tiles (cp.async, two stages, one chunk ahead).
#include "kmb_delta.cuh"

namespace kmb {
namespace {

template <int DKP, typename IO, bool KEEP>
__global__ void __launch_bounds__(128, 2)
delta_chain_fwd_kernel(const __grid_constant__ DeltaDesc d, int nw) {
    constexpr int C = kDeltaC;
    constexpr bool F32 = sizeof(IO) == 4;
    constexpr int NPK = F32 ? 2 : 1;
    constexpr int NPO = (F32 || KEEP) ? 2 : 1;   // pieces behind o: it is rounded to bf16 unless it is kept in fp32
    using ST = DeltaStage<C, DKP, NPK, NPO>;
    constexpr int NT = C / 8, KT = DKP / 8;
    constexpr int PK = C * DKP * 2;              // bytes of a K or Q piece
    extern __shared__ __align__(128) unsigned char sm[];
    const uint32_t sb = (uint32_t)__cvta_generic_to_shared(sm);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ub = (d.units + nw - 1) / nw;
    const int u = (int)(blockIdx.x % ub) * nw + warp;
    const int hv = (int)(blockIdx.x / ub) % d.Hv, n = (int)(blockIdx.x / ub) / d.Hv;
    const bool on = u < d.units;            // warps past dv only help with the copies
    const int r = lane >> 2, c2 = (lane & 3) * 2;
    const int col[2] = {u * 16 + r, u * 16 + r + 8};
    const bool cok[2] = {on && col[0] < d.dv, on && col[1] < d.dv};
    const int ldv = (int)d.ld_v, ldo = (int)d.ld_o;
    long long start, len;
    seq_range(d, n, start, len);
    const int chunk0 = d.cu ? d.cstart[n] : n * d.nc;
    const int nch = (int)((len + C - 1) / C);

    float S[KT][4];
    const size_t sbase = ((size_t)n * d.Hv + hv) * d.dk * d.dv;
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = t * 8 + c2 + (e & 1);
            S[t][e] = (d.h0 && i < d.dk && cok[e >> 1]) ? d.h0[sbase + (size_t)i * d.dv + col[e >> 1]] : 0.0f;
        }

    if (nch > 0) ST::load(d, d.Mt, sb, chunk0, hv);
    cp_commit();
    for (int c = 0; c < nch; c++) {
        if (c + 1 < nch) ST::load(d, d.Mt, sb + ((c + 1) & 1) * ST::BYTES, chunk0 + c + 1, hv);
        cp_commit();
        const long long tok0 = start + (long long)c * C;
        const int cnt = (int)(len - (long long)c * C < C ? len - (long long)c * C : C);
        // v of this chunk as accumulator tiles [16 columns][C tokens]; in flight under the first product
        float V[NT][4];
        {
            const IO* pv = (const IO*)d.v + tok0 * d.ld_v + (long long)hv * d.dv + col[0];
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + c2 + (e & 1);
                    V[t][e] = (i < cnt && cok[e >> 1]) ? ldt(pv + (long long)i * ldv, (e >> 1) * 8) : 0.0f;
                }
        }
        cp_wait<1>();
        __syncthreads();
        const uint32_t st = sb + (c & 1) * ST::BYTES;
        const float* tk = (const float*)(sm + (c & 1) * ST::BYTES + ST::oTok);
        const size_t fb = (((size_t)(chunk0 + c) * d.Hv + hv) * d.units + u);
        if (on) {
            if (KEEP) {
                float4* p = (float4*)d.Sf + fb * KT * 32 + lane;
#pragma unroll
                for (int t = 0; t < KT; t++) p[t * 32] = make_float4(S[t][0], S[t][1], S[t][2], S[t][3]);
            }
            float X[NT][4], O[NT][4], up[2], dn[2];
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) X[t][e] = O[t][e] = 0.0f;
            frag_scale(S, up, dn);
            const float sd[2] = {dn[0], dn[1]};
            if (KEEP) {
                const float m = warp_down(dn);
                if (lane == 0) d.mx[fb * MX_ROWS + MX_S] = m;
            }
#pragma unroll
            for (int kk = 0; kk < DKP / 16; kk++) {
                uint32_t a[2][4];
                frag_pieces<2>(S[2 * kk], S[2 * kk + 1], up, a);
                const auto ldk = [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4(b, st + p * PK + wide_off<C>(t2 * 16 + lb_row(lane), kk * 16 + lb_col(lane)));
                };
                const auto ldq = [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4(b, st + ST::oQ + p * PK + wide_off<C>(t2 * 16 + lb_row(lane), kk * 16 + lb_col(lane)));
                };
                mma_row<2, NPK>(X, a, 0, C / 16, ldk);
                mma_row<NPO, NPK>(O, reinterpret_cast<const uint32_t (&)[NPO][4]>(a), 0, C / 16, ldq);
            }
            // right-hand side v - e^gamma K S, and e^gamma Q S
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + c2 + (e & 1);
                    const float eg = tk[TOK_EG * C + i] * dn[e >> 1];
                    X[t][e] = V[t][e] - eg * tk[TOK_FK * C + i] * X[t][e];
                    O[t][e] *= eg * tk[TOK_FQ * C + i];
                }
            // W^T = X M^T: row i of M reaches columns j <= i only
            float U[NT][4];
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) U[t][e] = 0.0f;
            frag_scale(X, up, dn);
#pragma unroll
            for (int kk = 0; kk < C / 16; kk++) {
                uint32_t a[2][4];
                frag_pieces<2>(X[2 * kk], X[2 * kk + 1], up, a);
                mma_row<2, 2>(U, a, kk, C / 16, [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4(b, st + ST::oT + p * ST::TT + tile_off<C>(t2 * 16 + lb_row(lane), kk * 16 + lb_col(lane)));
                });
            }
            const float ft = tk[TOK_MISC * C], fp = tk[TOK_MISC * C + 1];
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) U[t][e] *= ft * dn[e >> 1];
            if (KEEP) {
                float4* p = (float4*)d.Wf + fb * NT * 32 + lane;
#pragma unroll
                for (int t = 0; t < NT; t++) p[t * 32] = make_float4(U[t][0], U[t][1], U[t][2], U[t][3]);
            }
            // U = beta W
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    U[t][e] *= tk[TOK_BETA * C + t * 8 + c2 + (e & 1)];
                    X[t][e] = 0.0f;
                }
            // O^T += U^T P^T
            frag_scale(U, up, dn);
            if (KEEP) {
                const float m = warp_down(dn);
                if (lane == 0) d.mx[fb * MX_ROWS + MX_U] = m;
            }
#pragma unroll
            for (int kk = 0; kk < C / 16; kk++) {
                uint32_t a[NPO][4];
                frag_pieces<NPO>(U[2 * kk], U[2 * kk + 1], up, a);
                mma_row<NPO, NPO>(X, a, kk, C / 16, [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4(b, st + ST::oP + p * ST::TT + tile_off<C>(t2 * 16 + lb_row(lane), kk * 16 + lb_col(lane)));
                });
            }
            IO* po = (IO*)d.o + tok0 * d.ld_o + (long long)hv * d.dv + col[0];
#pragma unroll
            for (int t = 0; t < NT; t++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + c2 + (e & 1);
                    O[t][e] = d.scale * fmaf(X[t][e], fp * dn[e >> 1], O[t][e]);
                    if (i < cnt && cok[e >> 1]) stt(po + (long long)i * ldo, (e >> 1) * 8, O[t][e]);
                }
                if (KEEP) *((float4*)d.Of + (fb * NT + t) * 32 + lane) = make_float4(O[t][0], O[t][1], O[t][2], O[t][3]);
            }
            // S^T <- e^gamma_C S^T + (G_C. U)^T K
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + c2 + (e & 1);
                    U[t][e] *= tk[TOK_GC * C + i] * tk[TOK_FK * C + i];
                }
            // The state takes the scale of U for the product and comes back after it (powers of two).  A U below
            // 2^-40 of the state is scaled as if it were that large, so the state does not overflow.
            const float last = tk[TOK_EG * C + C - 1];
            frag_scale(U, up, dn, sd[0] * last * kStateFloor, sd[1] * last * kStateFloor);
            const float s0 = last * up[0], s1 = last * up[1];
#pragma unroll
            for (int t = 0; t < KT; t++) {
                S[t][0] *= s0; S[t][1] *= s0;
                S[t][2] *= s1; S[t][3] *= s1;
            }
#pragma unroll
            for (int kk = 0; kk < C / 16; kk++) {
                uint32_t a[2][4];
                frag_pieces<2>(U[2 * kk], U[2 * kk + 1], up, a);
                mma_row<2, NPK>(S, a, 0, DKP / 16, [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4t(b, st + p * PK + wide_off<C>(kk * 16 + la_row(lane), t2 * 16 + la_col(lane)));
                });
            }
#pragma unroll
            for (int t = 0; t < KT; t++) {
                S[t][0] *= dn[0]; S[t][1] *= dn[0];
                S[t][2] *= dn[1]; S[t][3] *= dn[1];
            }
        }
        __syncthreads();   // the stage is free for the chunk after the next
    }
    if (d.hT) {
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = t * 8 + c2 + (e & 1);
                if (i < d.dk && cok[e >> 1]) d.hT[sbase + (size_t)i * d.dv + col[e >> 1]] = S[t][e];
            }
    }
    cp_wait<0>();
}

template <int DKP, typename IO, bool KEEP>
cudaError_t go(const DeltaDesc& d, cudaStream_t st) {
    constexpr bool F32 = sizeof(IO) == 4;
    using ST = DeltaStage<kDeltaC, DKP, F32 ? 2 : 1, (F32 || KEEP) ? 2 : 1>;
    const int nw = delta_warps(d);
    auto kern = delta_chain_fwd_kernel<DKP, IO, KEEP>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * ST::BYTES);
    if (e != cudaSuccess) return e;
    const long long blocks = (long long)d.nseq * d.Hv * ((d.units + nw - 1) / nw);
    kern<<<(unsigned)blocks, 32 * nw, 2 * ST::BYTES, st>>>(d, nw);
    return cudaGetLastError();
}
template <typename IO>
cudaError_t pick(const DeltaDesc& d, int DKP, bool keep, cudaStream_t st) {
    if (DKP == 64) return keep ? go<64, IO, true>(d, st) : go<64, IO, false>(d, st);
    return keep ? go<128, IO, true>(d, st) : go<128, IO, false>(d, st);
}
}  // namespace

cudaError_t delta_chain_fwd(const DeltaDesc& d, int DKP, bool bf16, bool keep, cudaStream_t st) {
    return bf16 ? pick<__nv_bfloat16>(d, DKP, keep, st) : pick<float>(d, DKP, keep, st);
}
}  // namespace kmb
