// delta.cu -- gated delta rule (include/kmamba_delta.h): entry points, the
// per-chunk matrices that need no state, and the recurrent form.
#include <cmath>
#include <cstring>
#include <initializer_list>
#include "kmb_delta.cuh"
#include "kmb_launch.cuh"
#include "../../include/kmamba_delta.h"

namespace kmb {
int set_error(const char* msg);
int set_cuda_error(const char* where, cudaError_t e);
void clear_error();
int* device_status();

namespace {

// ------------------------------------------------------------------ packed sequences
constexpr int kSortSeqs = 512;   // beyond that many sequences no single one matters
// One block: offsets clamped to [0, total] and made non-decreasing (cu), and the first chunk of each sequence
// (cstart).  Whatever the caller's offsets hold, the kernels stay inside the tensors.
__global__ void __launch_bounds__(256) delta_cu_kernel(const int* __restrict__ in, int nseq, int total, int C,
                                                       int* __restrict__ cu, int* __restrict__ cstart,
                                                       int* __restrict__ order) {
    pdl_release();
    __shared__ int sh[256], len[kSortSeqs];
    const int t = threadIdx.x;
    const int per = (nseq + 1 + 255) / 256;
    const int a = min(t * per, nseq + 1), b = min(a + per, nseq + 1);
    int mx = 0;
    for (int i = a; i < b; i++) mx = max(mx, min(max(in[i], 0), total));
    sh[t] = mx;
    __syncthreads();
    for (int o = 1; o < 256; o <<= 1) {
        const int v = t >= o ? sh[t - o] : 0;
        __syncthreads();
        sh[t] = max(sh[t], v);
        __syncthreads();
    }
    int run = t ? sh[t - 1] : 0;
    __syncthreads();
    for (int i = a; i < b; i++) {
        run = max(run, min(max(in[i], 0), total));
        cu[i] = run;
    }
    __threadfence_block();
    __syncthreads();
    int n = 0;   // chunks of sequences a .. b - 1
    for (int i = a; i < b && i < nseq; i++) n += (cu[i + 1] - cu[i] + C - 1) / C;
    sh[t] = n;
    __syncthreads();
    for (int o = 1; o < 256; o <<= 1) {
        const int v = t >= o ? sh[t - o] : 0;
        __syncthreads();
        sh[t] += v;
        __syncthreads();
    }
    n = t ? sh[t - 1] : 0;
    for (int i = a; i < b; i++) {
        cstart[i] = n;
        if (i < nseq) n += (cu[i + 1] - cu[i] + C - 1) / C;
    }
    // the longest sequences first, so that none of them starts last (ranks by counting; ties keep their order)
    if (nseq > kSortSeqs) return;
    for (int i = t; i < nseq; i += 256) len[i] = cu[i + 1] - cu[i];
    __syncthreads();
    for (int i = t; i < nseq; i += 256) {
        int rank = 0;
        for (int j = 0; j < nseq; j++) rank += len[j] > len[i] || (len[j] == len[i] && j < i);
        order[rank] = i;
    }
}

// ------------------------------------------------------------------ per-chunk matrices
// First K and Q as swizzled fp16 tiles (zero behind the last token and behind dk), each row with a power of two, per
// chunk and key head.  Then, per chunk and value head, four warps of 16 rows: K K^T and Q K^T, the token factors, P,
// and the chunk's triangular system.  With a_ij = G_ij k_i.k_j (j < i) and
//   C = (I + a diag(beta))^-1 a:   M = I - C diag(beta),   T = I - diag(beta) C
// (no division: both are exact where beta is 0).  By blocks of 16, diagonal blocks by forward substitution, one
// column per lane, then row block after row block
//   C_IJ = M_II (a_IJ - sum_{J <= K < I} a_IK diag(beta_K) C_KJ)
// on fp16 pieces: a warp holds its rows of a as accumulators, which are A fragments, and reads the finished C_K
// from shared memory.  Bound by latency (each row block waits for the last): what hides it is other blocks, so
// registers are held to four blocks per SM (100 us for 4096 chunks and heads of 64; three blocks: 108, five spill:
// 106), and tiles are a launch of their own (23 us, read and write bound).

template <int DKP, typename IO>
__global__ void __launch_bounds__(128)
delta_tiles_kernel(const __grid_constant__ DeltaDesc d, int vec) {
    constexpr int C = kDeltaC;
    constexpr bool F32 = sizeof(IO) == 4;
    constexpr int NPK = F32 ? 2 : 1;
    constexpr int TILE = C * DKP * 2;                     // bytes of one piece
    constexpr int G8 = DKP / 8;                           // threads per row of the tiles
    const int chunk = blockIdx.x, hk = blockIdx.y;
    long long tok0;
    int cnt;
    pdl_release();
    pdl_wait();   // the packed offsets
    if (!chunk_range<C>(d, chunk, tok0, cnt)) return;
    float* kf = d.kf + ((size_t)chunk * d.Hk + hk) * 2 * C;

    char* gK = (char*)(d.Kt + ((size_t)chunk * d.Hk + hk) * NPK * C * DKP);
    char* gQ = (char*)(d.Qt + ((size_t)chunk * d.Hk + hk) * NPK * C * DKP);
    // all loads of a batch are in flight before the first is used
    constexpr int NIT = 2 * C * G8 / 128, BATCH = F32 ? 4 : 8, V4 = F32 ? 2 : 1;
    for (int it0 = 0; it0 < NIT; it0 += BATCH) {
        uint4 raw[BATCH][V4];
        const auto place = [&](int it, bool& isq, int& row, int& c8) {
            const int i = it * 128 + threadIdx.x;
            isq = i >= C * G8;
            const int j = isq ? i - C * G8 : i;
            row = j / G8;
            c8 = j % G8 * 8;
            return isq ? (const IO*)d.q + (tok0 + row) * d.ld_q + (long long)hk * d.dk
                       : (const IO*)d.k + (tok0 + row) * d.ld_k + (long long)hk * d.dk;
        };
        if (vec) {
#pragma unroll
            for (int b = 0; b < BATCH; b++) {
                bool isq;
                int row, c8;
                const IO* src = place(it0 + b, isq, row, c8);
#pragma unroll
                for (int x = 0; x < V4; x++)
                    raw[b][x] = row < cnt && c8 + 8 <= d.dk ? *(const uint4*)(src + c8 + x * 4) : make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
            bool isq;
            int row, c8;
            const IO* src = place(it0 + b, isq, row, c8);
            float x[8];
            if (vec && (c8 + 8 <= d.dk || c8 >= d.dk)) {
#pragma unroll
                for (int v = 0; v < V4; v++) {
                    const uint32_t w[4] = {raw[b][v].x, raw[b][v].y, raw[b][v].z, raw[b][v].w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if constexpr (F32) {
                            x[v * 4 + e] = __uint_as_float(w[e]);
                        } else {
                            x[2 * e] = __uint_as_float(w[e] << 16);
                            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = row < cnt && c8 + e < d.dk ? ldt(src, c8 + e) : 0.0f;
            }
            float m = 0.0f, up, down;
#pragma unroll
            for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf(x[e]));
#pragma unroll
            for (int o = 1; o < G8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            row_scale(m, up, down);
            if (c8 == 0) kf[(isq ? C : 0) + row] = down;
            uint32_t w[4][NPK];
#pragma unroll
            for (int e = 0; e < 4; e++) split_pair<NPK>(x[2 * e] * up, x[2 * e + 1] * up, w[e]);
            const uint32_t o = wide_off<C>(row, c8);
#pragma unroll
            for (int k = 0; k < NPK; k++) {
                const uint4 p = make_uint4(w[0][k], w[1][k], w[2][k], w[3][k]);
                *(uint4*)((isq ? gQ : gK) + k * TILE + o) = p;
            }
        }
    }
}

template <int DKP, int NPK>
__global__ void __launch_bounds__(128, DKP * NPK <= 128 ? 4 : 3)
delta_prep_kernel(const __grid_constant__ DeltaDesc d, int train) {
    constexpr int C = kDeltaC;
    constexpr int TILE = C * DKP * 2;                     // bytes of one piece
    constexpr int TT = C * C * 2;
    extern __shared__ __align__(128) unsigned char sm[];
    const uint32_t sK = (uint32_t)__cvta_generic_to_shared(sm), sQ = sK + NPK * TILE;
    unsigned char* Csm = sm;                              // C, two pieces, in the place of K and Q
    __shared__ double gam[C];
    __shared__ float rowE[C], colE[3 * 48], bet[C], fK[C], fQ[C], fC[4];
    __shared__ float dg[4][16][17];                       // diagonal blocks, per warp
    __shared__ __align__(128) unsigned char Ysm[2 * 16 * 128];   // the row block in work, two pieces
    const DecaySmem dec{gam, rowE, colE};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int chunk = blockIdx.x, hv = blockIdx.y, hk = hv / d.grp;
    long long tok0;
    int cnt;
    pdl_release();
    if (d.cu) pdl_wait();   // the packed offsets
    if (!chunk_range<C>(d, chunk, tok0, cnt)) return;
    float g2[2], b2[2];     // gates: tokens lane and lane + 32
    if (warp < 2) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int i = h * 32 + lane;
            const long long at = (tok0 + i) * d.Hv + hv;
            g2[h] = (warp == 0 && d.g && i < cnt) ? d.g[at] : 0.0f;
            b2[h] = (warp == 1 && i < cnt) ? (d.beta ? d.beta[at] : 1.0f) : 0.0f;
        }
    }
    if (!d.cu) pdl_wait();
    {
        const char* gK = (const char*)(d.Kt + ((size_t)chunk * d.Hk + hk) * NPK * C * DKP);
        const char* gQ = (const char*)(d.Qt + ((size_t)chunk * d.Hk + hk) * NPK * C * DKP);
#pragma unroll 4
        for (int i = threadIdx.x; i < NPK * TILE / 16; i += 128) {
            cp16(sK + i * 16, gK + i * 16);
            cp16(sQ + i * 16, gQ + i * 16);
        }
        cp_commit();
    }
    const size_t head = (size_t)chunk * d.Hv + hv;
    float* tk = d.tok + head * TOK_SIZE;
    if (warp == 0) {
        running_sums(g2[0], g2[1], lane, gam);
        __syncwarp();
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int i = h * 32 + lane;
            if (train) d.gam[head * C + i] = gam[i];
            tk[TOK_EG * C + i] = expf((float)gam[i]);
            tk[TOK_GC * C + i] = expf((float)(gam[C - 1] - gam[i]));
        }
    } else if (warp == 1) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int i = h * 32 + lane;
            bet[i] = b2[h];
            tk[TOK_BETA * C + i] = b2[h];
        }
    } else {
        const float* kf = d.kf + ((size_t)chunk * d.Hk + hk) * 2 * C;
        const int i = threadIdx.x - 64;
        const float k = kf[i], q = kf[C + i];
        fK[i] = k;
        fQ[i] = q;
        tk[TOK_FK * C + i] = k;
        tk[TOK_FQ * C + i] = q;
    }
    cp_wait<0>();
    __syncthreads();
    decay_tables(dec, threadIdx.x);
    const int rg = warp;
    const int r = lane >> 2, c2 = (lane & 3) * 2;
    float A[C / 8][4], B[C / 8][4];   // K K^T and Q K^T, columns up to the diagonal block; then a and P
    zero(A);
    zero(B);
#pragma unroll
    for (int s = 0; s < DKP / 16; s++) {
        uint32_t ak[NPK][4], aq[NPK][4];
        const uint32_t oa = wide_off<C>(rg * 16 + la_row(lane), s * 16 + la_col(lane));
#pragma unroll
        for (int p = 0; p < NPK; p++) {
            ldm4(ak[p], sK + p * TILE + oa);
            ldm4(aq[p], sQ + p * TILE + oa);
        }
#pragma unroll
        for (int t2 = 0; t2 < C / 16; t2++) {
            if (t2 > rg) continue;
            uint32_t b[NPK][4];
#pragma unroll
            for (int p = 0; p < NPK; p++)
                ldm4(b[p], sK + p * TILE + wide_off<C>(t2 * 16 + lb_row(lane), s * 16 + lb_col(lane)));
#pragma unroll
            for (int pb = 0; pb < NPK; pb++)
#pragma unroll
                for (int pa = 0; pa + pb < NPK; pa++) {
                    mma(A[2 * t2], ak[pa], b[pb][0], b[pb][1]);
                    mma(A[2 * t2 + 1], ak[pa], b[pb][2], b[pb][3]);
                    mma(B[2 * t2], aq[pa], b[pb][0], b[pb][1]);
                    mma(B[2 * t2 + 1], aq[pa], b[pb][2], b[pb][3]);
                }
        }
    }
    __syncthreads();   // the tables are there, K and Q are read
    {
        const uint32_t sC = sK, sY = (uint32_t)__cvta_generic_to_shared(Ysm);
        // rows of a and P on and below the warp's diagonal block
        float pm = 0.0f;
#pragma unroll
        for (int t = 0; t < C / 8; t++) {
            if ((t >> 1) > rg) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = rg * 16 + r + (e >> 1) * 8, j = t * 8 + c2 + (e & 1);
                const float G = dec.at(i, j, (t >> 1) == rg, rg) * fK[j];
                B[t][e] *= G * fQ[i];
                pm = fmaxf(pm, fabsf(B[t][e]));
                A[t][e] = j < i ? A[t][e] * (G * fK[i]) : 0.0f;
            }
        }
        float up, down;
        warp_scale(pm, up, down);
        if (lane == 0) tk[TOK_MISC * C + 4 + rg] = down;
        const auto put = [&](char* g, const float (&x)[C / 8][4], float s, bool shared) {
#pragma unroll
            for (int t = 0; t < C / 8; t++) {
                if ((t >> 1) > rg) continue;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t p[2];
                    split_pair<2>(x[t][h * 2] * s, x[t][h * 2 + 1] * s, p);
                    const uint32_t o = tile_off<C>(rg * 16 + r + h * 8, t * 8 + c2);
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        if (shared) *(uint32_t*)(Csm + k * TT + o) = p[k];
                        if (g) *(uint32_t*)(g + k * TT + o) = p[k];
                    }
                }
            }
        };
        put((char*)(d.Pt + head * 2 * C * C), B, up, false);
        // C_II: the diagonal block through shared memory, column `lane` of the solution, back as accumulator tiles
#pragma unroll
        for (int t = 0; t < C / 8; t++)
            if ((t >> 1) == rg) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    dg[warp][r + (e >> 1) * 8][(t & 1) * 8 + c2 + (e & 1)] = A[t][e];
                    A[t][e] = 0.0f;
                }
            }
        __syncwarp();
        {
            float x[16], xb[16];   // the column, and beta times it
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float s = dg[warp][i][lane & 15];
#pragma unroll
                for (int j = 0; j < i; j++) s = fmaf(-dg[warp][i][j], xb[j], s);
                x[i] = s;
                xb[i] = s * bet[warp * 16 + i];
            }
            __syncwarp();
            if (lane < 16) {
#pragma unroll
                for (int i = 0; i < 16; i++) dg[warp][i][lane] = x[i];
            }
            __syncwarp();
        }
        float S[C / 8][4], md[2][4];   // the warp's rows of C; M_II
#pragma unroll
        for (int t = 0; t < C / 8; t++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                S[t][e] = (t >> 1) == rg ? dg[warp][r + (e >> 1) * 8][(t & 1) * 8 + c2 + (e & 1)] : 0.0f;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = r + (e >> 1) * 8, j = t * 8 + c2 + (e & 1);
                md[t][e] = (i == j ? 1.0f : 0.0f) - dg[warp][i][j] * bet[warp * 16 + j];
            }
        for (int I = 0; I < 4; I++) {
            if (warp == I) {
                if (I > 0) {
                    float Y[6][4], aup, adn, part[6][4];
#pragma unroll
                    for (int t = 0; t < 6; t++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            Y[t][e] = A[t][e];
                            A[t][e] *= bet[t * 8 + c2 + (e & 1)];
                        }
                    frag_scale(A, aup, adn);
#pragma unroll
                    for (int K = 0; K < 3; K++) {
                        if (K >= I) continue;
                        uint32_t a[2][4];
                        frag_pieces<2>(A[2 * K], A[2 * K + 1], aup, a);
                        zero(part);
                        mma_row<2, 2>(part, a, 0, K + 1, [&](int p, int t2, uint32_t (&b)[4]) {
                            ldm4t(b, sC + p * TT + tile_off<C>(K * 16 + la_row(lane), t2 * 16 + la_col(lane)));
                        });
                        add_scaled(Y, part, -adn * fC[K]);
                    }
                    float yu, ym;
                    frag_scale(Y, yu, ym);
#pragma unroll
                    for (int t = 0; t < 6; t++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            uint32_t p[2];
                            split_pair<2>(Y[t][h * 2] * yu, Y[t][h * 2 + 1] * yu, p);
                            const uint32_t o = tile_off<C>(r + h * 8, t * 8 + c2);
#pragma unroll
                            for (int k = 0; k < 2; k++) *(uint32_t*)(Ysm + k * 2048 + o) = p[k];
                        }
                    __syncwarp();
                    uint32_t a[2][4];
                    frag_scale(md, aup, adn);
                    frag_pieces<2>(md[0], md[1], aup, a);
                    zero(part);
                    mma_row<2, 2>(part, a, 0, 3, [&](int p, int t2, uint32_t (&b)[4]) {
                        ldm4t(b, sY + p * 2048 + tile_off<C>(la_row(lane), t2 * 16 + la_col(lane)));
                    });
#pragma unroll
                    for (int t = 0; t < 6; t++)
                        if ((t >> 1) < rg) {
#pragma unroll
                            for (int e = 0; e < 4; e++) S[t][e] = part[t][e] * (adn * ym);
                        }
                }
                if (I < 3) {
                    float cu, cm;
                    frag_scale(S, cu, cm);
                    if (lane == 0) fC[I] = cm;
                    put(nullptr, S, cu, true);
                }
            }
            __syncthreads();
        }
        // T = I - diag(beta) C, M = I - C diag(beta): the warp's rows, one power of two each
        float tm = 0.0f, mm = 0.0f;
#pragma unroll
        for (int t = 0; t < C / 8; t++) {
            if ((t >> 1) > rg) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = rg * 16 + r + (e >> 1) * 8, j = t * 8 + c2 + (e & 1);
                const float one = i == j ? 1.0f : 0.0f;
                A[t][e] = one - bet[i] * S[t][e];
                S[t][e] = one - S[t][e] * bet[j];
                tm = fmaxf(tm, fabsf(A[t][e]));
                mm = fmaxf(mm, fabsf(S[t][e]));
            }
        }
        warp_scale(mm, up, down);
        if (lane == 0) tk[TOK_MISC * C + rg] = down;
        put((char*)(d.Mt + head * 2 * C * C), S, up, false);
        if (train) {
            warp_scale(tm, up, down);
            if (lane == 0) tk[TOK_MISC * C + 8 + rg] = down;
            put((char*)(d.Tt + head * 2 * C * C), A, up, false);
        }
    }
}

template <int DKP, typename IO>
cudaError_t prep_go(const DeltaDesc& d, int train, cudaStream_t st) {
    constexpr int C = kDeltaC, NPK = sizeof(IO) == 4 ? 2 : 1;
    constexpr int kq = 2 * NPK * C * DKP * 2, cc = 2 * C * C * 2, sm = kq > cc ? kq : cc;
    auto kern = delta_prep_kernel<DKP, NPK>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, sm);
    if (e != cudaSuccess) return e;
    const int V = 16 / (int)sizeof(IO);
    const int vec = d.dk % V == 0 && d.ld_q % V == 0 && d.ld_k % V == 0 && ((uintptr_t)d.q & 15) == 0 &&
                    ((uintptr_t)d.k & 15) == 0;
    e = launch(delta_tiles_kernel<DKP, IO>, dim3((unsigned)d.nch, (unsigned)d.Hk), dim3(128), 0, st, d.cu != nullptr, d,
               vec);
    if (e != cudaSuccess) return e;
    return launch(kern, dim3((unsigned)d.nch, (unsigned)d.Hv), dim3(128), sm, st, true, d, train);
}

// ------------------------------------------------------------------ recurrent form
// A warp owns 16 columns of one head's state, all dk rows: lane = 8 row groups x 4 groups of 4 columns, NR rows
// per lane, so the state is read and written once in 16-byte pieces and stays in registers for the T tokens.
// Per token two sums over dk (k.S and q.S), each a chain over the lane's rows and three shuffles.  Bound by the
// state's bytes: 8 dk dv of them a head.  Measured: 250 rows of 16 heads of 128 x 128 in 93 us, 5.6 TB/s of the
// states' bytes (87 % of a copy's rate); 102 us with keys and queries read entry by entry at three blocks per SM.
struct StepDesc {
    long long batch, T;
    int Hk, Hv, grp, dk, dv, units;
    float scale;
    const void *q, *k, *v;
    const float *g, *beta;
    void* o;
    long long ld_q, ld_k, ld_v, ld_o;
    float* pool;
    long long n_slots;
    const int* slots;
};

// The lane's NR entries of a token's key or query
template <typename IO, int NR>
struct StepRow {
    static constexpr int N4 = NR * (int)sizeof(IO) / 16;
    uint4 w[N4];
    __device__ __forceinline__ void load(const IO* p, int r0, int dk, bool vec) {
        if (vec) {   // dk is a multiple of 16 bytes: whole pieces are inside or outside
#pragma unroll
            for (int i = 0; i < N4; i++)
                w[i] = r0 + i * (16 / (int)sizeof(IO)) < dk ? *(const uint4*)(p + r0 + i * (16 / (int)sizeof(IO)))
                                                            : make_uint4(0, 0, 0, 0);
        } else {
            alignas(16) IO e[NR];
#pragma unroll
            for (int i = 0; i < NR; i++) {
                if (r0 + i < dk) e[i] = p[r0 + i];
                else stt(e, i, 0.0f);
            }
#pragma unroll
            for (int i = 0; i < N4; i++) w[i] = ((const uint4*)e)[i];
        }
    }
    __device__ __forceinline__ float get(int i) const {
        const uint32_t* u = (const uint32_t*)w;
        if constexpr (sizeof(IO) == 4) return __uint_as_float(u[i]);
        else return __uint_as_float((i & 1) ? u[i >> 1] & 0xffff0000u : u[i >> 1] << 16);
    }
};

// four blocks of four warps per SM: 128 registers, of which the state takes 64
template <typename IO, int NR, bool VEC>
__global__ void __launch_bounds__(128, NR == 16 ? 4 : 6)
delta_step_kernel(const __grid_constant__ StepDesc d, int vec) {
    const int lane = threadIdx.x & 31;
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (id >= d.batch * d.Hv * d.units) return;
    const int u = (int)(id % d.units), hv = (int)(id / d.units % d.Hv);
    const long long b = id / d.units / d.Hv;
    const int hk = hv / d.grp, rl = lane >> 2, cl = lane & 3;
    const int c0 = u * 16 + cl * 4, r0 = rl * NR;
    const long long slot = d.slots ? d.slots[b] : b;
    const IO *q = (const IO*)d.q, *k = (const IO*)d.k, *v = (const IO*)d.v;
    IO* o = (IO*)d.o;
    if (slot < 0 || slot >= d.n_slots) {
        for (long long t = 0; t < d.T; t++)
            for (int e = 0; e < 4; e++)
                if (rl == 0 && c0 + e < d.dv) stt(o, (b * d.T + t) * d.ld_o + (long long)hv * d.dv + c0 + e, 0.0f);
        return;
    }
    float* Sg = d.pool + ((size_t)slot * d.Hv + hv) * d.dk * d.dv;
    float S[NR][4];
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int row = r0 + i;
        if (VEC && row < d.dk && c0 < d.dv) {
            const float4 x = *(const float4*)(Sg + (size_t)row * d.dv + c0);
            S[i][0] = x.x; S[i][1] = x.y; S[i][2] = x.z; S[i][3] = x.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) S[i][e] = row < d.dk && c0 + e < d.dv ? Sg[(size_t)row * d.dv + c0 + e] : 0.0f;
        }
    }
    for (long long t = 0; t < d.T; t++) {
        const long long tok = b * d.T + t;
        const float al = d.g ? expf(d.g[tok * d.Hv + hv]) : 1.0f;
        const float be = d.beta ? d.beta[tok * d.Hv + hv] : 1.0f;
        StepRow<IO, NR> kr, qr;
        float vc[4];
        kr.load(k + tok * d.ld_k + (long long)hk * d.dk, r0, d.dk, vec);
        qr.load(q + tok * d.ld_q + (long long)hk * d.dk, r0, d.dk, vec);
#pragma unroll
        for (int e = 0; e < 4; e++)
            vc[e] = c0 + e < d.dv ? ldt(v, tok * d.ld_v + (long long)hv * d.dv + c0 + e) : 0.0f;
        if (al == 0.0f) {   // forgotten, whatever it holds (0 times an infinity or NaN would stay one)
#pragma unroll
            for (int i = 0; i < NR; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) S[i][e] = 0.0f;
        }
        float p[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NR; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                S[i][e] *= al;
                p[e] = fmaf(S[i][e], kr.get(i), p[e]);
            }
#pragma unroll
        for (int s = 4; s < 32; s <<= 1)
#pragma unroll
            for (int e = 0; e < 4; e++) p[e] += __shfl_xor_sync(0xffffffffu, p[e], s);
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 4; e++) p[e] = be * (vc[e] - p[e]);
#pragma unroll
        for (int i = 0; i < NR; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                S[i][e] = fmaf(kr.get(i), p[e], S[i][e]);
                y[e] = fmaf(S[i][e], qr.get(i), y[e]);
            }
#pragma unroll
        for (int s = 4; s < 32; s <<= 1)
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] += __shfl_xor_sync(0xffffffffu, y[e], s);
        if (rl == 0) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (c0 + e < d.dv) stt(o, tok * d.ld_o + (long long)hv * d.dv + c0 + e, d.scale * y[e]);
        }
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int row = r0 + i;
        if (VEC && row < d.dk && c0 < d.dv) {
            *(float4*)(Sg + (size_t)row * d.dv + c0) = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (row < d.dk && c0 + e < d.dv) Sg[(size_t)row * d.dv + c0 + e] = S[i][e];
        }
    }
}
template <typename IO>
cudaError_t step_go(const StepDesc& d, cudaStream_t st) {
    const long long warps = d.batch * d.Hv * d.units;
    const unsigned blocks = (unsigned)((warps + 3) / 4);
    const bool vec = d.dv % 4 == 0 && ((uintptr_t)d.pool & 15) == 0;
    const int V = 16 / (int)sizeof(IO);
    const int vkq = d.dk % V == 0 && d.ld_q % V == 0 && d.ld_k % V == 0 && ((uintptr_t)d.q & 15) == 0 &&
                    ((uintptr_t)d.k & 15) == 0;
    if (d.dk <= 64) {
        if (vec) delta_step_kernel<IO, 8, true><<<blocks, 128, 0, st>>>(d, vkq);
        else delta_step_kernel<IO, 8, false><<<blocks, 128, 0, st>>>(d, vkq);
    } else {
        if (vec) delta_step_kernel<IO, 16, true><<<blocks, 128, 0, st>>>(d, vkq);
        else delta_step_kernel<IO, 16, false><<<blocks, 128, 0, st>>>(d, vkq);
    }
    return cudaGetLastError();
}

// ------------------------------------------------------------------ host
const char* check(const KMBDeltaParams* p) {
    if (!p) return "delta: null parameters";
    if (p->batch < 0 || p->T < 0) return "delta: batch and T must be >= 0";
    if (p->Hk < 1 || p->Hv < 1 || p->Hv % p->Hk) return "delta: Hv must be a positive multiple of Hk";
    if (p->Hk > 65535 || p->Hv > 65535) return "delta: at most 65535 heads";
    if (p->dk < 1 || p->dv < 1 || p->dk > KMB_DELTA_MAX_DIM || p->dv > KMB_DELTA_MAX_DIM)
        return "delta: dk and dv must be in 1 .. 128";
    if (p->dtype != KMB_DTYPE_F32 && p->dtype != KMB_DTYPE_BF16) return "delta: unknown dtype";
    if (p->cu_seqlens) {
        if (p->batch != 1 || p->n_seq < 1) return "delta: packed sequences need batch = 1 and n_seq >= 1";
        if (p->n_seq > (1L << 24)) return "delta: at most 2^24 packed sequences";
    }
    if (p->batch > (1L << 24) || p->T > 0x7fffffc0L || (double)p->batch * (double)p->T > 2147483584.0)
        return "delta: at most 2^31 - 64 tokens";
    if ((p->ld_q && p->ld_q < p->Hk * p->dk) || (p->ld_k && p->ld_k < p->Hk * p->dk) ||
        (p->ld_v && p->ld_v < p->Hv * p->dv) || (p->ld_o && p->ld_o < p->Hv * p->dv))
        return "delta: a token stride is shorter than a token";
    if (p->ld_q > 0x7fffffffL || p->ld_k > 0x7fffffffL || p->ld_v > 0x7fffffffL || p->ld_o > 0x7fffffffL)
        return "delta: a token stride is at most 2^31 - 1 elements";
    return nullptr;
}
// whether one of the pointers is off its element's boundary (an access there is an error of the device)
bool off(size_t size, std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if ((uintptr_t)p % size) return true;
    return false;
}
constexpr const char* kOff = "delta: a tensor is not aligned to its elements";
size_t elem(const KMBDeltaParams* p) { return p->dtype == KMB_DTYPE_BF16 ? 2 : 4; }
bool off(const KMBDeltaParams* p) {
    return off(elem(p), {p->q, p->k, p->v, p->o}) || off(4, {p->g, p->beta, p->h0, p->hT, p->cu_seqlens});
}
const char* check_launch(const KMBDeltaParams* p, const DeltaDesc& d) {
    if ((double)d.nseq * d.Hv * d.units > 2147483647.0) return "delta: too many sequences times heads for one launch";
    if ((double)d.nch * d.Hv > 2147483647.0) return "delta: too many chunks times heads for one launch";
    (void)p;
    return nullptr;
}

// Shapes, pieces and workspace of a call; returns the workspace's bytes
size_t layout(const KMBDeltaParams* p, bool train, float* ws, DeltaDesc& d, int& DKP) {
    constexpr int C = kDeltaC;
    memset(&d, 0, sizeof d);
    DKP = p->dk <= 64 ? 64 : 128;
    const int NPK = p->dtype == KMB_DTYPE_BF16 ? 1 : 2;
    d.T = p->T;
    d.total = p->batch * p->T;
    d.nseq = p->cu_seqlens ? (int)p->n_seq : (int)p->batch;
    d.cu_in = p->cu_seqlens;
    d.nc = (int)((p->T + C - 1) / C);
    d.nch = p->cu_seqlens ? (int)(p->T / C + p->n_seq) : (int)(p->batch * d.nc);
    d.Hk = (int)p->Hk; d.Hv = (int)p->Hv; d.grp = d.Hv / d.Hk; d.dk = (int)p->dk; d.dv = (int)p->dv;
    d.units = (d.dv + 15) / 16;
    d.scale = p->scale;
    d.q = p->q; d.k = p->k; d.v = p->v; d.g = p->g; d.beta = p->beta; d.h0 = p->h0; d.o = p->o; d.hT = p->hT;
    d.ld_q = p->ld_q ? p->ld_q : p->Hk * p->dk;
    d.ld_k = p->ld_k ? p->ld_k : p->Hk * p->dk;
    d.ld_v = p->ld_v ? p->ld_v : p->Hv * p->dv;
    d.ld_o = p->ld_o ? p->ld_o : p->Hv * p->dv;
    size_t o = 0;
    char* base = (char*)ws;
    auto take = [&](size_t bytes) {
        char* r = base + o;
        o += (bytes + 127) & ~(size_t)127;
        return r;
    };
    if (p->cu_seqlens) {
        d.cu = (const int*)take((size_t)(d.nseq + 1) * 4);
        d.cstart = (const int*)take((size_t)(d.nseq + 1) * 4);
        if (d.nseq <= kSortSeqs) d.order = (const int*)take((size_t)d.nseq * 4);
    }
    const size_t ck = (size_t)d.nch * d.Hk, cv = (size_t)d.nch * d.Hv;
    d.Kt = (__half*)take(ck * NPK * C * DKP * 2);
    d.Qt = (__half*)take(ck * NPK * C * DKP * 2);
    d.Mt = (__half*)take(cv * 2 * C * C * 2);
    d.Pt = (__half*)take(cv * 2 * C * C * 2);
    d.kf = (float*)take(ck * 2 * C * 4);
    d.tok = (float*)take(cv * TOK_SIZE * 4);
    if (train) {
        const size_t u = cv * d.units * 16 * 2;   // bytes of a column of a unit's tile
        d.Tt = (__half*)take(cv * 2 * C * C * 2);
        d.gam = (double*)take(cv * C * 8);
        d.Sh = (__half*)take(u * 2 * DKP);
        d.Sf = (float*)take(u * 2 * DKP);
        d.Wh = (__half*)take(u * 2 * C);
        d.Of = (float*)take(u * 2 * C);
        d.Wf = (float*)take(u * 2 * C);
        d.Rf = (float*)take(u * 2 * C);
        d.Gh = (__half*)take(u * NPK * C);
        d.Rh = (__half*)take(u * 2 * C);
        d.dSh = (__half*)take(u * 2 * DKP);
        d.anchor = (float*)take(cv * d.units * 4 * 4);
        d.mx = (float*)take(cv * d.units * 4 * MX_ROWS * 4);
    }
    return o;
}

}  // namespace

int delta_sms() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n;
}

static cudaError_t delta_prep(const DeltaDesc& d, int DKP, bool bf16, int train, cudaStream_t st) {
    if (bf16)
        return DKP == 64 ? prep_go<64, __nv_bfloat16>(d, train, st) : prep_go<128, __nv_bfloat16>(d, train, st);
    return DKP == 64 ? prep_go<64, float>(d, train, st) : prep_go<128, float>(d, train, st);
}

}  // namespace kmb

using namespace kmb;

extern "C" {

size_t kmb_delta_workspace_floats(const KMBDeltaParams* p, int train) {
    if (check(p)) return 0;
    DeltaDesc d;
    int DKP;
    return (layout(p, train != 0, nullptr, d, DKP) + 3) / 4;
}

int kmb_delta_forward(const KMBDeltaParams* p, float* ws, int keep, void* stream) {
    clear_error();
    if (const char* m = check(p)) return set_error(m);
    DeltaDesc d;
    int DKP;
    layout(p, keep != 0, ws, d, DKP);
    if (d.nseq == 0) return 0;
    if (d.total > 0 && (!p->q || !p->k || !p->v || !p->o)) return set_error("delta: q, k, v and o are required");
    if (off(p)) return set_error(kOff);
    if (!ws || ((uintptr_t)ws & 15)) return set_error("delta: a 16-byte aligned workspace is required");
    if (const char* m = check_launch(p, d)) return set_error(m);
    const bool bf16 = p->dtype == KMB_DTYPE_BF16;
    cudaStream_t st = (cudaStream_t)stream;
    d.status = device_status();
    cudaError_t e = cudaSuccess;
    if (d.cu) {
        delta_cu_kernel<<<1, 256, 0, st>>>(d.cu_in, d.nseq, (int)d.total, kDeltaC, (int*)d.cu, (int*)d.cstart, (int*)d.order);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess && d.nch > 0) e = delta_prep(d, DKP, bf16, keep != 0, st);
    if (e == cudaSuccess) e = delta_chain_fwd(d, DKP, bf16, keep != 0, st);
    return e == cudaSuccess ? 0 : set_cuda_error("kmb_delta_forward", e);
}

int kmb_delta_backward(const KMBDeltaParams* p, const KMBDeltaGrads* g, float* ws, void* stream) {
    clear_error();
    if (const char* m = check(p)) return set_error(m);
    if (!g) return set_error("delta backward: null gradients");
    DeltaDesc d;
    int DKP;
    layout(p, true, ws, d, DKP);
    if (d.nseq == 0) return 0;
    if (d.total > 0 && (!p->q || !p->k || !p->v || !g->do_ || !g->dq || !g->dk || !g->dv))
        return set_error("delta backward: q, k, v, do, dq, dk and dv are required");
    if ((g->ld_do && g->ld_do < p->Hv * p->dv) || (g->ld_dq && g->ld_dq < p->Hk * p->dk) ||
        (g->ld_dk && g->ld_dk < p->Hk * p->dk) || (g->ld_dv && g->ld_dv < p->Hv * p->dv))
        return set_error("delta backward: a token stride is shorter than a token");
    if (g->ld_do > 0x7fffffffL || g->ld_dq > 0x7fffffffL || g->ld_dk > 0x7fffffffL || g->ld_dv > 0x7fffffffL)
        return set_error("delta backward: a token stride is at most 2^31 - 1 elements");
    if (off(p) || off(elem(p), {g->do_, g->dq, g->dk, g->dv}) || off(4, {g->dhT, g->dg, g->dbeta, g->dh0}))
        return set_error(kOff);
    if (!ws || ((uintptr_t)ws & 15)) return set_error("delta backward: the forward's workspace is required");
    if (const char* m = check_launch(p, d)) return set_error(m);
    d.go = g->do_; d.dhT = g->dhT; d.dq = g->dq; d.dkk = g->dk; d.dvv = g->dv;
    d.dg = g->dg; d.dbeta = g->dbeta; d.dh0 = g->dh0;
    d.ld_do = g->ld_do ? g->ld_do : p->Hv * p->dv;
    d.ld_dq = g->ld_dq ? g->ld_dq : p->Hk * p->dk;
    d.ld_dk = g->ld_dk ? g->ld_dk : p->Hk * p->dk;
    d.ld_dv = g->ld_dv ? g->ld_dv : p->Hv * p->dv;
    const bool bf16 = p->dtype == KMB_DTYPE_BF16;
    cudaStream_t st = (cudaStream_t)stream;
    d.status = device_status();
    cudaError_t e = delta_chain_bwd(d, DKP, bf16, st);
    if (e == cudaSuccess && d.nch > 0) e = delta_grads(d, DKP, bf16, st);
    return e == cudaSuccess ? 0 : set_cuda_error("kmb_delta_backward", e);
}

int kmb_delta_step(const KMBDeltaParams* p, float* pool, long n_slots, const int* slots, void* stream) {
    clear_error();
    if (const char* m = check(p)) return set_error(m);
    if (p->cu_seqlens || p->h0 || p->hT) return set_error("kmb_delta_step: cu_seqlens, h0 and hT must be NULL");
    if (p->batch == 0 || p->T == 0) return 0;
    if (!p->q || !p->k || !p->v || !p->o || !pool) return set_error("kmb_delta_step: q, k, v, o and the pool are required");
    if (n_slots < 0) return set_error("kmb_delta_step: n_slots must be >= 0");
    if (off(p) || off(4, {pool, slots})) return set_error(kOff);
    StepDesc d{};
    d.batch = p->batch; d.T = p->T; d.Hk = (int)p->Hk; d.Hv = (int)p->Hv; d.grp = d.Hv / d.Hk;
    d.dk = (int)p->dk; d.dv = (int)p->dv; d.units = (d.dv + 15) / 16; d.scale = p->scale;
    if ((double)d.batch * d.Hv * d.units > 4.0 * 2147483647.0) return set_error("kmb_delta_step: batch times heads is too large");
    d.q = p->q; d.k = p->k; d.v = p->v; d.g = p->g; d.beta = p->beta; d.o = p->o;
    d.ld_q = p->ld_q ? p->ld_q : p->Hk * p->dk;
    d.ld_k = p->ld_k ? p->ld_k : p->Hk * p->dk;
    d.ld_v = p->ld_v ? p->ld_v : p->Hv * p->dv;
    d.ld_o = p->ld_o ? p->ld_o : p->Hv * p->dv;
    d.pool = pool; d.n_slots = n_slots; d.slots = slots;
    cudaError_t e = p->dtype == KMB_DTYPE_BF16 ? step_go<__nv_bfloat16>(d, (cudaStream_t)stream)
                                               : step_go<float>(d, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : set_cuda_error("kmb_delta_step", e);
}

}  // extern "C"
