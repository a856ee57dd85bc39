// delta_bwd.cu -- gated delta rule, backward.
//
// With the chunk's T and P (kmb_delta.cuh) the adjoint is, from the last chunk
// to the first,
//   dU = scale P^T dO + diag(G_C.) K dS_C;   dR = T^T dU;   dV = beta dR
//   dS_0 = e^gamma_C dS_C + scale (e^gamma Q)^T dO - (beta e^gamma K)^T dR
// the forward's three products again, run the other way by the same scheme (a
// warp owns 16 columns of dv and keeps dS^T in registers).  All else has no
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
// over dv of what the recurrence holds in fp32.
#include "kmb_delta.cuh"

namespace kmb {
namespace {

template <int DKP, typename IO>
__global__ void __launch_bounds__(128, 2)
delta_chain_bwd_kernel(const __grid_constant__ DeltaDesc d, int nw) {
    constexpr int C = kDeltaC;
    constexpr bool F32 = sizeof(IO) == 4;
    constexpr int NPK = F32 ? 2 : 1;
    using ST = DeltaStage<C, DKP, NPK, 2>;
    constexpr int NT = C / 8, KT = DKP / 8;
    constexpr int PK = C * DKP * 2;
    extern __shared__ __align__(128) unsigned char sm[];
    const uint32_t sb = (uint32_t)__cvta_generic_to_shared(sm);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ub = (d.units + nw - 1) / nw;
    const int u = (int)(blockIdx.x % ub) * nw + warp;
    const int hv = (int)(blockIdx.x / ub) % d.Hv, n = (int)(blockIdx.x / ub) / d.Hv;
    const bool on = u < d.units;
    const int r = lane >> 2, c2 = (lane & 3) * 2;
    const int col[2] = {u * 16 + r, u * 16 + r + 8};
    const bool cok[2] = {on && col[0] < d.dv, on && col[1] < d.dv};
    const int ldv = (int)d.ld_v, ldo = (int)d.ld_do, lddv = (int)d.ld_dv;
    long long start, len;
    seq_range(d, n, start, len);
    const int chunk0 = d.cu ? d.cstart[n] : n * d.nc;
    const int nch = (int)((len + C - 1) / C);

    float S[KT][4];   // dS^T
    const size_t sbase = ((size_t)n * d.Hv + hv) * d.dk * d.dv;
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = t * 8 + c2 + (e & 1);
            S[t][e] = (d.dhT && i < d.dk && cok[e >> 1]) ? d.dhT[sbase + (size_t)i * d.dv + col[e >> 1]] : 0.0f;
        }

    if (nch > 0) ST::load(d, d.Tt, sb, chunk0 + nch - 1, hv);
    cp_commit();
    for (int it = 0; it < nch; it++) {
        const int c = nch - 1 - it;
        if (c > 0) ST::load(d, d.Tt, sb + ((it + 1) & 1) * ST::BYTES, chunk0 + c - 1, hv);
        cp_commit();
        const long long tok0 = start + (long long)c * C;
        const int cnt = (int)(len - (long long)c * C < C ? len - (long long)c * C : C);
        const size_t fb = (((size_t)(chunk0 + c) * d.Hv + hv) * d.units + u);
        float G[NT][4];   // dO^T
        {
            const IO* p = (const IO*)d.go + tok0 * d.ld_do + (long long)hv * d.dv + col[0];
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + c2 + (e & 1);
                    G[t][e] = (i < cnt && cok[e >> 1]) ? ldt(p + (long long)i * ldo, (e >> 1) * 8) : 0.0f;
                }
        }
        cp_wait<1>();
        __syncthreads();
        const uint32_t st = sb + (it & 1) * ST::BYTES;
        const float* tk = (const float*)(sm + (it & 1) * ST::BYTES + ST::oTok);
        if (on) {
            float X[NT][4], Y[NT][4], up[2], dn[2], ts[NT][2], bs[NT][2];
#pragma unroll
            for (int t = 0; t < NT; t++) {
#pragma unroll
                for (int e = 0; e < 4; e++) X[t][e] = Y[t][e] = 0.0f;
                ts[t][0] = ts[t][1] = bs[t][0] = bs[t][1] = 0.0f;
            }
            // K dS_C
            frag_scale(S, up, dn);
            const float sd[2] = {dn[0], dn[1]};
            {
                const float m = warp_down(dn);
                if (lane == 0) d.mx[fb * MX_ROWS + MX_DS] = m;
                float4* p = (float4*)d.dSf + fb * KT * 32 + lane;
#pragma unroll
                for (int t = 0; t < KT; t++) p[t * 32] = make_float4(S[t][0], S[t][1], S[t][2], S[t][3]);
            }
#pragma unroll
            for (int kk = 0; kk < DKP / 16; kk++) {
                uint32_t a[2][4];
                frag_pieces<2>(S[2 * kk], S[2 * kk + 1], up, a);
                mma_row<2, NPK>(X, a, 0, C / 16, [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4(b, st + p * PK + wide_off<C>(t2 * 16 + lb_row(lane), kk * 16 + lb_col(lane)));
                });
            }
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + c2 + (e & 1);
                    X[t][e] *= tk[TOK_GC * C + i] * tk[TOK_FK * C + i] * dn[e >> 1];
                }
            // P^T dO: column j of P has rows i >= j only
            frag_scale(G, up, dn);
            {
                const float m = warp_down(dn);
                if (lane == 0) d.mx[fb * MX_ROWS + MX_DO] = m;
            }
#pragma unroll
            for (int kk = 0; kk < C / 16; kk++) {
                uint32_t a[NPK][4];
                frag_pieces<NPK>(G[2 * kk], G[2 * kk + 1], up, a);
                mma_row<NPK, 2>(Y, a, 0, kk + 1, [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4t(b, st + ST::oP + p * ST::TT + tile_off<C>(kk * 16 + la_row(lane), t2 * 16 + la_col(lane)));
                });
            }
            const float ft = tk[TOK_MISC * C + 2], fp = tk[TOK_MISC * C + 1] * d.scale;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    X[t][e] = fmaf(Y[t][e], fp * dn[e >> 1], X[t][e]);
                    Y[t][e] = 0.0f;
                }
            // dR^T = dU^T T
            frag_scale(X, up, dn);
#pragma unroll
            for (int kk = 0; kk < C / 16; kk++) {
                uint32_t a[2][4];
                frag_pieces<2>(X[2 * kk], X[2 * kk + 1], up, a);
                mma_row<2, 2>(Y, a, 0, kk + 1, [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4t(b, st + ST::oT + p * ST::TT + tile_off<C>(kk * 16 + la_row(lane), t2 * 16 + la_col(lane)));
                });
            }
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) Y[t][e] *= ft * dn[e >> 1];
            frag_scale(Y, up, dn);
            {
                const float m = warp_down(dn);
                if (lane == 0) d.mx[fb * MX_ROWS + MX_R] = m;
            }
            // dV, and what the gates' gradients sum over dv
            {
                const float4* pu = (const float4*)d.Wf + fb * NT * 32 + lane;
                const float4* po = (const float4*)d.Of + fb * NT * 32 + lane;
                float4* pr = (float4*)d.Rf + fb * NT * 32 + lane;
                const IO* pv = (const IO*)d.v + tok0 * d.ld_v + (long long)hv * d.dv + col[0];
                IO* pd = (IO*)d.dvv + tok0 * d.ld_dv + (long long)hv * d.dv + col[0];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const float4 u4 = pu[t * 32], o4 = po[t * 32];
                    pr[t * 32] = make_float4(Y[t][0], Y[t][1], Y[t][2], Y[t][3]);
                    const float uu[4] = {u4.x, u4.y, u4.z, u4.w}, oo[4] = {o4.x, o4.y, o4.z, o4.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int i = t * 8 + c2 + (e & 1);
                        const float dv = tk[TOK_BETA * C + i] * Y[t][e];
                        bs[t][e & 1] = fmaf(Y[t][e], uu[e], bs[t][e & 1]);
                        ts[t][e & 1] = fmaf(G[t][e], oo[e], ts[t][e & 1]);
                        if (i < cnt && cok[e >> 1]) {
                            ts[t][e & 1] = fmaf(-ldt(pv + (long long)i * ldv, (e >> 1) * 8), dv, ts[t][e & 1]);
                            stt(pd + (long long)i * lddv, (e >> 1) * 8, dv);
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) {
                            ts[t][h] += __shfl_xor_sync(0xffffffffu, ts[t][h], o);
                            bs[t][h] += __shfl_xor_sync(0xffffffffu, bs[t][h], o);
                        }
                float* pp = d.part + fb * 2 * C;
#pragma unroll
                for (int t = 0; t < NT; t++)
                    if (r == t) {
                        pp[t * 8 + c2] = ts[t][0];
                        pp[t * 8 + c2 + 1] = ts[t][1];
                        pp[C + t * 8 + c2] = bs[t][0];
                        pp[C + t * 8 + c2 + 1] = bs[t][1];
                    }
            }
            // dS^T <- e^gamma_C dS^T + (scale e^gamma dO)^T Q - (beta e^gamma dR)^T K, one scale per row for both
            const float last = tk[TOK_EG * C + C - 1];
            float m0 = sd[0] * last * kStateFloor, m1 = sd[1] * last * kStateFloor;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = t * 8 + c2 + (e & 1);
                    const float eg = tk[TOK_EG * C + i];
                    G[t][e] *= d.scale * eg * tk[TOK_FQ * C + i];
                    Y[t][e] *= -tk[TOK_BETA * C + i] * eg * tk[TOK_FK * C + i];
                    if (e < 2) m0 = fmaxf(m0, fabsf(G[t][e]));
                    else m1 = fmaxf(m1, fabsf(G[t][e]));
                }
            frag_scale(Y, up, dn, m0, m1);
            const float s0 = last * up[0], s1 = last * up[1];
#pragma unroll
            for (int t = 0; t < KT; t++) {
                S[t][0] *= s0; S[t][1] *= s0;
                S[t][2] *= s1; S[t][3] *= s1;
            }
#pragma unroll
            for (int kk = 0; kk < C / 16; kk++) {
                uint32_t a[2][4];
                frag_pieces<2>(G[2 * kk], G[2 * kk + 1], up, a);
                mma_row<2, NPK>(S, a, 0, DKP / 16, [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4t(b, st + ST::oQ + p * PK + wide_off<C>(kk * 16 + la_row(lane), t2 * 16 + la_col(lane)));
                });
                frag_pieces<2>(Y[2 * kk], Y[2 * kk + 1], up, a);
                mma_row<2, NPK>(S, a, 0, DKP / 16, [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4t(b, st + p * PK + wide_off<C>(kk * 16 + la_row(lane), t2 * 16 + la_col(lane)));
                });
            }
            // <S_0, dS_0> over the warp's columns
            float an = 0.0f;
            const float4* ps = (const float4*)d.Sf + fb * KT * 32 + lane;
#pragma unroll
            for (int t = 0; t < KT; t++) {
                S[t][0] *= dn[0]; S[t][1] *= dn[0];
                S[t][2] *= dn[1]; S[t][3] *= dn[1];
                const float4 x = ps[t * 32];
                an = fmaf(S[t][0], x.x, an);
                an = fmaf(S[t][1], x.y, an);
                an = fmaf(S[t][2], x.z, an);
                an = fmaf(S[t][3], x.w, an);
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) an += __shfl_xor_sync(0xffffffffu, an, o);
            if (lane == 0) d.anchor[fb] = an;
        }
        __syncthreads();
    }
    if (d.dh0) {
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = t * 8 + c2 + (e & 1);
                if (i < d.dk && cok[e >> 1]) d.dh0[sbase + (size_t)i * d.dv + col[e >> 1]] = S[t][e];
            }
    }
    cp_wait<0>();
}

// ------------------------------------------------------------------ gradients without recurrence
// Eight warps: 16 token rows x half of dk (and half of the 64 columns of dP, dA) each.  dv is walked in slices of
// 64, staged as fp16 tiles in one piece (bf16 results: 11 bits are enough before the rounding) or two (fp32); a
// tile has one power of two, from the largest entry that the recurrences recorded.
template <int DKP, int NP>
struct GradSmem {
    static constexpr int C = kDeltaC;
    static constexpr int KQ = NP * C * DKP * 2, T64 = 64 * C * 2, SD = 64 * DKP * 2;
    static constexpr int oK = 0, oQ = KQ, oG = 2 * KQ, oU = oG + NP * T64, oR = oU + NP * T64, oS = oR + NP * T64,
                         oD = oS + NP * SD, oEnd = oD + NP * SD;
    // the four weighted matrices take the place of the slices
    static constexpr int oE = oG, TE = C * C * 2;
    static constexpr int oTok = (oE + 4 * NP * TE > oEnd ? oE + 4 * NP * TE : oEnd);
    static constexpr int oGam = oTok + TOK_ROWS * C * 4;
    static constexpr int BYTES = oGam + C * 8;
};

// 2^14-based scale of the largest of the units' records
__device__ __forceinline__ void units_scale(const float* mx, int units, int which, float& up, float& down) {
    float m = 0.0f;
    for (int i = 0; i < units; i++) m = fmaxf(m, mx[i * MX_ROWS + which]);
    down = m;
    up = 1.0f / m;   // a power of two, at least 2^-126
}

template <int DKP, typename IO>
__global__ void __launch_bounds__(256, 1)
delta_grads_kernel(const __grid_constant__ DeltaDesc d, int vec) {
    constexpr int C = kDeltaC;
    constexpr bool F32 = sizeof(IO) == 4;
    constexpr int NP = F32 ? 2 : 1;
    using SM = GradSmem<DKP, NP>;
    constexpr int HN = DKP / 2, HT = HN / 8, KT = DKP / 8, NT = C / 8;
    constexpr int PK = C * DKP * 2;
    extern __shared__ __align__(128) unsigned char sm[];
    __shared__ float red[4][8];
    const uint32_t sb = (uint32_t)__cvta_generic_to_shared(sm);
    float* tk = (float*)(sm + SM::oTok);
    double* gam = (double*)(sm + SM::oGam);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rg = warp & 3, ch = warp >> 2;
    const int r = lane >> 2, c2 = (lane & 3) * 2;
    const int chunk = blockIdx.x, hk = blockIdx.y;
    long long tok0;
    int cnt;
    if (!chunk_range<C>(d, chunk, tok0, cnt)) return;
    {
        const char* ks = (const char*)(d.Kt + ((size_t)chunk * d.Hk + hk) * NP * C * DKP);
        const char* qs = (const char*)(d.Qt + ((size_t)chunk * d.Hk + hk) * NP * C * DKP);
        for (int i = tid; i < SM::KQ / 16; i += 256) {
            cp16(sb + SM::oK + i * 16, ks + i * 16);
            cp16(sb + SM::oQ + i * 16, qs + i * 16);
        }
        cp_commit();
    }
    float dQ[HT][4], dK[HT][4];
#pragma unroll
    for (int t = 0; t < HT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) dQ[t][e] = dK[t][e] = 0.0f;

    for (int hh = 0; hh < d.grp; hh++) {
        const int hv = hk * d.grp + hh;
        const size_t head = (size_t)chunk * d.Hv + hv;
        __syncthreads();
        for (int i = tid; i < TOK_ROWS * C; i += 256) tk[i] = d.tok[head * TOK_ROWS * C + i];
        if (warp == 0) {
            double carry = 0.0;
#pragma unroll
            for (int h = 0; h < C / 32; h++) {
                const int i = h * 32 + lane;
                float g = (d.g && i < cnt) ? d.g[(tok0 + i) * d.Hv + hv] : 0.0f;
                if (g < -104.0f) g = -104.0f;
                double s = g;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double t = __shfl_up_sync(0xffffffffu, s, o);
                    if (lane >= o) s += t;
                }
                s += carry;
                gam[i] = s;
                carry = __shfl_sync(0xffffffffu, s, 31);
            }
        } else if (warp == 1 && (d.dg || d.dbeta)) {
            // gates: tokens lane and lane + 32
            double before = 0.0, anchor = 0.0;
            for (int x = 0; x < d.units; x++) anchor += d.anchor[head * d.units + x];
#pragma unroll
            for (int h = 0; h < C / 32; h++) {
                const int i = h * 32 + lane;
                double t = 0.0;
                float b = 0.0f;
                for (int x = 0; x < d.units; x++) {
                    t += d.part[((head * d.units + x) * 2) * C + i];
                    b += d.part[((head * d.units + x) * 2 + 1) * C + i];
                }
                double s = t;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double y = __shfl_up_sync(0xffffffffu, s, o);
                    if (lane >= o) s += y;
                }
                if (i < cnt) {
                    const long long at = (tok0 + i) * d.Hv + hv;
                    // a decay below e^-104 is 0 in fp32: nothing depends on it
                    const bool reset = d.g && d.g[at] < -104.0f;
                    if (d.dg) d.dg[at] = reset ? 0.0f : (float)(anchor - (before + s - t));
                    if (d.dbeta) d.dbeta[at] = b;
                }
                before += __shfl_sync(0xffffffffu, s, 31);
            }
        }
        const float* mx = d.mx + head * d.units * MX_ROWS;
        float uS, sS, uU, sU, uG, sG, uR, sR, uD, sD;
        units_scale(mx, d.units, MX_S, uS, sS);
        units_scale(mx, d.units, MX_U, uU, sU);
        units_scale(mx, d.units, MX_DO, uG, sG);
        units_scale(mx, d.units, MX_R, uR, sR);
        units_scale(mx, d.units, MX_DS, uD, sD);

        float dP[4][4], dA[4][4], q1[HT][4], z1[HT][4], k1[HT][4];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) dP[t][e] = dA[t][e] = 0.0f;
#pragma unroll
        for (int t = 0; t < HT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) q1[t][e] = z1[t][e] = k1[t][e] = 0.0f;

        for (int u0 = 0; u0 < d.units; u0 += 4) {
            __syncthreads();
            // dO: [tokens][64 columns]
            for (int i = tid; i < C * 8; i += 256) {
                const int row = i >> 3, c8 = (i & 7) * 8, cc = u0 * 16 + c8;
                const IO* src = (const IO*)d.go + (tok0 + row) * d.ld_do + (long long)hv * d.dv + cc;
                float x[8];
                if (vec && row < cnt && cc + 8 <= d.dv) {
                    if constexpr (F32) {
                        const float4 a = *(const float4*)src, b = *(const float4*)(src + 4);
                        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
                        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
                    } else {
                        const uint4 a = *(const uint4*)src;
                        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            x[2 * e] = __uint_as_float(w[e] << 16);
                            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
                        }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = row < cnt && cc + e < d.dv ? ldt(src, e) : 0.0f;
                }
                uint32_t w[4][NP];
#pragma unroll
                for (int e = 0; e < 4; e++) split_pair<NP>(x[2 * e] * uG, x[2 * e + 1] * uG, w[e]);
#pragma unroll
                for (int k = 0; k < NP; k++)
                    *(uint4*)(sm + SM::oG + k * SM::T64 + tile_off<64>(row, c8)) =
                        make_uint4(w[0][k], w[1][k], w[2][k], w[3][k]);
            }
            // U, dR: [64 columns of dv][tokens]
            for (int i = tid; i < 4 * NT * 32; i += 256) {
                const int x = i / (NT * 32), t = i / 32 % NT, l = i & 31;
                float4 uu = make_float4(0.0f, 0.0f, 0.0f, 0.0f), rr = uu;
                if (u0 + x < d.units) {
                    const size_t at = ((head * d.units + u0 + x) * NT + t) * 32 + l;
                    uu = ((const float4*)d.Wf)[at];
                    rr = ((const float4*)d.Rf)[at];
                }
                const int tok = t * 8 + (l & 3) * 2, row = x * 16 + (l >> 2);
                const float a0 = tk[TOK_BETA * C + tok] * uU, a1 = tk[TOK_BETA * C + tok + 1] * uU;
                uint32_t p[NP], q[NP];
                const uint32_t o0 = tile_off<64>(row, tok), o1 = tile_off<64>(row + 8, tok);
                split_pair<NP>(uu.x * a0, uu.y * a1, p);
                split_pair<NP>(rr.x * uR, rr.y * uR, q);
#pragma unroll
                for (int k = 0; k < NP; k++) {
                    *(uint32_t*)(sm + SM::oU + k * SM::T64 + o0) = p[k];
                    *(uint32_t*)(sm + SM::oR + k * SM::T64 + o0) = q[k];
                }
                split_pair<NP>(uu.z * a0, uu.w * a1, p);
                split_pair<NP>(rr.z * uR, rr.w * uR, q);
#pragma unroll
                for (int k = 0; k < NP; k++) {
                    *(uint32_t*)(sm + SM::oU + k * SM::T64 + o1) = p[k];
                    *(uint32_t*)(sm + SM::oR + k * SM::T64 + o1) = q[k];
                }
            }
            // S_0, dS_C: [64 columns of dv][dk]
            for (int i = tid; i < 4 * KT * 32; i += 256) {
                const int x = i / (KT * 32), t = i / 32 % KT, l = i & 31;
                float4 ss = make_float4(0.0f, 0.0f, 0.0f, 0.0f), dd = ss;
                if (u0 + x < d.units) {
                    const size_t at = ((head * d.units + u0 + x) * KT + t) * 32 + l;
                    ss = ((const float4*)d.Sf)[at];
                    dd = ((const float4*)d.dSf)[at];
                }
                const int kc = t * 8 + (l & 3) * 2, row = x * 16 + (l >> 2);
                uint32_t p[NP], q[NP];
                const uint32_t o0 = wide_off<64>(row, kc), o1 = wide_off<64>(row + 8, kc);
                split_pair<NP>(ss.x * uS, ss.y * uS, p);
                split_pair<NP>(dd.x * uD, dd.y * uD, q);
#pragma unroll
                for (int k = 0; k < NP; k++) {
                    *(uint32_t*)(sm + SM::oS + k * SM::SD + o0) = p[k];
                    *(uint32_t*)(sm + SM::oD + k * SM::SD + o0) = q[k];
                }
                split_pair<NP>(ss.z * uS, ss.w * uS, p);
                split_pair<NP>(dd.z * uD, dd.w * uD, q);
#pragma unroll
                for (int k = 0; k < NP; k++) {
                    *(uint32_t*)(sm + SM::oS + k * SM::SD + o1) = p[k];
                    *(uint32_t*)(sm + SM::oD + k * SM::SD + o1) = q[k];
                }
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < 4; kk++) {
                uint32_t aG[NP][4], aR[NP][4], aU[NP][4];
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    ldm4(aG[p], sb + SM::oG + p * SM::T64 + tile_off<64>(rg * 16 + la_row(lane), kk * 16 + la_col(lane)));
                    ldm4t(aR[p], sb + SM::oR + p * SM::T64 + tile_off<64>(kk * 16 + lb_row(lane), rg * 16 + lb_col(lane)));
                    ldm4t(aU[p], sb + SM::oU + p * SM::T64 + tile_off<64>(kk * 16 + lb_row(lane), rg * 16 + lb_col(lane)));
                }
                const auto ldu = [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4t(b, sb + SM::oU + p * SM::T64 +
                                 tile_off<64>(kk * 16 + la_row(lane), ch * 32 + t2 * 16 + la_col(lane)));
                };
                if (ch * 2 <= rg) {   // columns above the diagonal blocks are not needed
                    mma_row<NP, NP>(dP, aG, 0, 2, ldu);
                    mma_row<NP, NP>(dA, aR, 0, 2, ldu);
                }
                const auto lds = [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4t(b, sb + SM::oS + p * SM::SD +
                                 wide_off<64>(kk * 16 + la_row(lane), ch * HN + t2 * 16 + la_col(lane)));
                };
                const auto ldd = [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4t(b, sb + SM::oD + p * SM::SD +
                                 wide_off<64>(kk * 16 + la_row(lane), ch * HN + t2 * 16 + la_col(lane)));
                };
                mma_row<NP, NP>(q1, aG, 0, HN / 16, lds);
                mma_row<NP, NP>(z1, aR, 0, HN / 16, lds);
                mma_row<NP, NP>(k1, aU, 0, HN / 16, ldd);
            }
        }
        // weighted matrices: E = scale G dO U^T with the key's and with the query's tile scale, F = -beta G dR U^T
        // with the key's of either side
        float m[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const float wP = d.scale * sG * sU, wA = -sR * sU;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = rg * 16 + r + (e >> 1) * 8, j = ch * 32 + t * 8 + c2 + (e & 1);
                const float g = j <= i ? expf((float)(gam[i] - gam[j])) : 0.0f;
                dP[t][e] = j <= i ? g * wP * dP[t][e] : 0.0f;
                dA[t][e] = j < i ? g * wA * tk[TOK_BETA * C + i] * dA[t][e] : 0.0f;
                m[0] = fmaxf(m[0], fabsf(dP[t][e] * tk[TOK_FK * C + j]));
                m[1] = fmaxf(m[1], fabsf(dP[t][e] * tk[TOK_FQ * C + i]));
                m[2] = fmaxf(m[2], fabsf(dA[t][e] * tk[TOK_FK * C + j]));
                m[3] = fmaxf(m[3], fabsf(dA[t][e] * tk[TOK_FK * C + i]));
            }
#pragma unroll
        for (int k = 0; k < 4; k++) {
#pragma unroll
            for (int o = 16; o; o >>= 1) m[k] = fmaxf(m[k], __shfl_xor_sync(0xffffffffu, m[k], o));
            if (lane == 0) red[k][warp] = m[k];
        }
        cp_wait<0>();
        __syncthreads();   // the slices are read, K and Q have arrived
        float eu[4], ed[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float x = red[k][0];
#pragma unroll
            for (int w = 1; w < 8; w++) x = fmaxf(x, red[k][w]);
            row_scale(x, eu[k], ed[k]);
        }
#pragma unroll
        for (int t = 0; t < 4; t++)
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
                    uint32_t p[NP];
                    split_pair<NP>(v[k][0] * eu[k], v[k][1] * eu[k], p);
#pragma unroll
                    for (int x = 0; x < NP; x++) *(uint32_t*)(sm + SM::oE + (k * NP + x) * SM::TE + o) = p[x];
                }
            }
        __syncthreads();
        // fold the products over dv into the sums, then the four products over tokens
        float fq[2], fz[2], fu[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int i = rg * 16 + r + h * 8;
            const float eg = tk[TOK_EG * C + i];
            fq[h] = d.scale * eg * sG * sS;
            fz[h] = -tk[TOK_BETA * C + i] * eg * sR * sS;
            fu[h] = tk[TOK_GC * C + i] * sU * sD;
        }
#pragma unroll
        for (int t = 0; t < HT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                dQ[t][e] = fmaf(fq[e >> 1], q1[t][e], dQ[t][e]);
                dK[t][e] = fmaf(fz[e >> 1], z1[t][e], dK[t][e]);
                dK[t][e] = fmaf(fu[e >> 1], k1[t][e], dK[t][e]);
            }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            // k: 0 E K -> dQ, 2 F K -> dK (rows i, sum over j <= i); 1 E^T Q, 3 F^T K -> dK (rows j, sum over i >= j)
            float acc[HT][4];
#pragma unroll
            for (int t = 0; t < HT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[t][e] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < C / 16; kk++) {
                if ((k & 1) ? kk < rg : kk > rg) continue;
                uint32_t a[NP][4];
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    const uint32_t base = sb + SM::oE + (k * NP + p) * SM::TE;
                    if (k & 1) ldm4t(a[p], base + tile_off<C>(kk * 16 + lb_row(lane), rg * 16 + lb_col(lane)));
                    else ldm4(a[p], base + tile_off<C>(rg * 16 + la_row(lane), kk * 16 + la_col(lane)));
                }
                mma_row<NP, NP>(acc, a, 0, HN / 16, [&](int p, int t2, uint32_t (&b)[4]) {
                    ldm4t(b, sb + (k == 1 ? SM::oQ : SM::oK) + p * PK +
                                 wide_off<C>(kk * 16 + la_row(lane), ch * HN + t2 * 16 + la_col(lane)));
                });
            }
#pragma unroll
            for (int t = 0; t < HT; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (k == 0) dQ[t][e] = fmaf(ed[k], acc[t][e], dQ[t][e]);
                    else dK[t][e] = fmaf(ed[k], acc[t][e], dK[t][e]);
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

template <int DKP, typename IO>
cudaError_t chain_go(const DeltaDesc& d, cudaStream_t st) {
    using ST = DeltaStage<kDeltaC, DKP, sizeof(IO) == 4 ? 2 : 1, 2>;
    const int nw = delta_warps(d);
    auto kern = delta_chain_bwd_kernel<DKP, IO>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * ST::BYTES);
    if (e != cudaSuccess) return e;
    const long long blocks = (long long)d.nseq * d.Hv * ((d.units + nw - 1) / nw);
    kern<<<(unsigned)blocks, 32 * nw, 2 * ST::BYTES, st>>>(d, nw);
    return cudaGetLastError();
}
template <int DKP, typename IO>
cudaError_t grads_go(const DeltaDesc& d, cudaStream_t st) {
    using SM = GradSmem<DKP, sizeof(IO) == 4 ? 2 : 1>;
    auto kern = delta_grads_kernel<DKP, IO>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::BYTES);
    if (e != cudaSuccess) return e;
    const int V = 16 / (int)sizeof(IO);
    const int vec = d.dv % V == 0 && d.ld_do % V == 0 && ((uintptr_t)d.go & 15) == 0;
    kern<<<dim3((unsigned)d.nch, (unsigned)d.Hk), 256, SM::BYTES, st>>>(d, vec);
    return cudaGetLastError();
}
}  // namespace

cudaError_t delta_chain_bwd(const DeltaDesc& d, int DKP, bool bf16, cudaStream_t st) {
    if (bf16) return DKP == 64 ? chain_go<64, __nv_bfloat16>(d, st) : chain_go<128, __nv_bfloat16>(d, st);
    return DKP == 64 ? chain_go<64, float>(d, st) : chain_go<128, float>(d, st);
}
cudaError_t delta_grads(const DeltaDesc& d, int DKP, bool bf16, cudaStream_t st) {
    if (bf16) return DKP == 64 ? grads_go<64, __nv_bfloat16>(d, st) : grads_go<128, __nv_bfloat16>(d, st);
    return DKP == 64 ? grads_go<64, float>(d, st) : grads_go<128, float>(d, st);
}
}  // namespace kmb
