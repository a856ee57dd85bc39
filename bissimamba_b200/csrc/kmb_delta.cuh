// kmb_delta.cuh -- shared pieces of the gated delta rule's kernels (delta.cu,
// delta_fwd.cu, delta_bwd.cu).
//
// Chunk of C tokens of one value head, gamma_i the running sum of g inside it,
// G_ij = exp(gamma_i - gamma_j):
//   w_i = v_i - e^gamma_i S_0^T k_i - sum_{j < i} G_ij (k_i.k_j) u_j,   u_i = beta_i w_i
//   O = scale (diag(e^gamma) Q S_0 + P U),   P_ij = G_ij q_i.k_j (j <= i)
//   S_C = e^gamma_C S_0 + sum_j G_Cj k_j u_j^T
// With a_ij = G_ij k_i.k_j (j < i):  W = M (V - diag(e^gamma) K S_0), M = (I + a diag(beta))^-1,
// and the adjoint of U is T^T dU, T = (I + diag(beta) a)^-1.  W and T^T dU are full where beta is 0, and their product
// is beta's gradient, so the forward takes M and the backward T.
// M, T and P depend on no state: a first kernel computes them for all chunks at
// once; the recurrence over chunks then is three products a chunk.
//
// Products run on mma.sync (fp16 factors, fp32 accumulation).  A row or a block of
// 16 of an fp32 factor is scaled by a power of two to a largest entry in
// [2^14, 2^15) and cut into two fp16 pieces x = x0 + x1, each rounded to nearest:
// 22 bits down to 2^-18 of the largest entry, and an absolute floor 2^-40 below
// it, so it holds what an fp32 product needs.  The three products x0 y0, x0 y1,
// x1 y0 are summed; a bf16 row is a single piece (8 bits fit in 11), everything
// computed is two, whatever type the result is rounded to.  Three bf16 pieces would
// take six products for the same accuracy.  The powers of two are undone in the fp32
// factors that multiply the accumulators anyway.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include "kmb_sync.cuh"

namespace kmb {

// rows of the token factors of a chunk and value head
enum {
    TOK_EG = 0,    // e^gamma_i
    TOK_GC = 1,    // G_Ci = exp(gamma_C - gamma_i)
    TOK_BETA = 2,  // beta, 0 behind the last token
    TOK_FK = 3,    // k_i = FK_i * row i of the K tile
    TOK_FQ = 4,
    TOK_MISC = 5,  // [b], [4 + b], [8 + b]: rows 16 b .. 16 b + 15 of M, P, T = that factor times their tiles
    TOK_SIZE = 5 * 64 + 16   // floats
};
enum { MX_S = 0, MX_W = 1, MX_DO = 2, MX_R = 3, MX_DS = 4, MX_ROWS = 8 };
constexpr int kDeltaC = 64;      // tokens per chunk

struct DeltaDesc {
    long long T, total;          // tokens per sequence (fixed length), tokens in all
    int nseq;
    const int* cu;               // ws: sanitised offsets [nseq + 1] (packed), else NULL
    const int* cstart;           // ws: first chunk of each sequence [nseq + 1] (packed)
    const int* cu_in;            // the caller's offsets
    int nch, nc;                 // chunks at most; chunks per sequence (fixed length)
    int Hk, Hv, grp, dk, dv, units;   // units: 16-column slices of dv
    float scale;
    const void *q, *k, *v;
    const float *g, *beta, *h0;
    void* o;
    float* hT;
    long long ld_q, ld_k, ld_v, ld_o;
    // workspace
    __half *Kt, *Qt;             // [nch][Hk][pieces][C * DKP] swizzled tiles, rows scaled
    __half *Mt, *Pt, *Tt;        // [nch][Hv][2][C * C], on and below the diagonal blocks; Tt for training only
    float* kf;                   // [nch][Hk][2][C]: what the rows of the K and of the Q tile are times
    float* tok;                  // [nch][Hv][TOK_SIZE], see TOK_*
    double* gam;                 // [nch][Hv][C]: running sums of g (training)
    const int* order;            // packed: sequences, the longest first (NULL: as they are)
    // kept for the backward, per unit: swizzled fp16 tiles of 16 rows (columns of dv), in pieces, each warp's part
    // scaled by a power of two (mx)
    __half *Sh, *Wh;             // state at the chunk's start [2][16 * DKP], W [2][16 * C]
    __half *Gh, *Rh, *dSh;       // backward: dO [pieces of v][16 * C], dR = T^T dU [2][16 * C], adjoint of the state at the end
    float *Sf, *Of, *Wf, *Rf;    // state, O, W and dR in accumulator order [tiles][32 lanes][4]
    float* anchor;               // [nch][Hv][units][4 warps]: <S_0, dS_0> of their parts
    float* mx;                   // [nch][Hv][units][4 warps][MX_ROWS]: what the tiles of S, W, dO, dR, dS are times
    // gradients
    const void* go;
    const float* dhT;
    void *dq, *dkk, *dvv;
    float *dg, *dbeta, *dh0;
    int* status;
    long long ld_do, ld_dq, ld_dk, ld_dv;
};

// 16-byte pieces of a row are XOR-swizzled by the row so that ldmatrix reads 8 rows without bank conflicts.
// Tiles are W = 64 or 32 columns wide; wider matrices are several 64-column tiles, `rows` * 128 bytes apart.
template <int W>
__device__ __forceinline__ uint32_t tile_off(int row, int col) {
    if (W == 64) return (uint32_t)(row * 128 + ((((col >> 3) ^ row) & 7) << 4) + ((col & 7) << 1));
    return (uint32_t)(row * 64 + ((((col >> 3) ^ (row >> 1)) & 3) << 4) + ((col & 7) << 1));
}
// matrix of `rows` rows and a multiple of 64 columns
template <int ROWS>
__device__ __forceinline__ uint32_t wide_off(int row, int col) {
    return (uint32_t)((col >> 6) * (ROWS * 128)) + tile_off<64>(row, col & 63);
}

__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// lane addresses of ldmatrix.x4, for a 16 x 16 block at (r0, c0):
//   as stored  -> A fragment a0..a3 (rows = m, columns = k)
__device__ __forceinline__ int la_row(int lane) { return (lane & 7) + ((lane >> 3) & 1) * 8; }
__device__ __forceinline__ int la_col(int lane) { return (lane >> 4) * 8; }
//   as stored  -> B fragments b0 b1 | b0 b1 of two n-tiles (rows = n, columns = k); with .trans and rows = m
//   (stored transposed, [k][m]) the A fragment takes the same addresses
__device__ __forceinline__ int lb_row(int lane) { return (lane & 7) + (lane >> 4) * 8; }
__device__ __forceinline__ int lb_col(int lane) { return ((lane >> 3) & 1) * 8; }
//   .trans, rows = k, columns = n -> B fragments of two n-tiles: la_row, la_col

// fp16 pieces of the pair (x, y), rounded to nearest
template <int NP>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&p)[NP]) {
    __half2 h = __floats2half2_rn(x, y);
    p[0] = *reinterpret_cast<const uint32_t*>(&h);
    if constexpr (NP == 2) {
        h = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
        p[1] = *reinterpret_cast<const uint32_t*>(&h);
    }
}
// Power of two that takes m (the largest magnitude of a row) into [2^14, 2^15), and its inverse.  Rows below
// 2^-112 (zero rows among them) take the factors of 2^-112.  Beside an infinity nothing finite would be left, so it
// makes the row NaN; a NaN entry stays one.
__device__ __forceinline__ void row_scale(float m, float& up, float& down) {
    int e = (int)(__float_as_uint(m) >> 23);
    e = e < 15 ? 15 : e;
    up = __uint_as_float(e == 255 ? 0x7fffffffu : (uint32_t)(268 - e) << 23);
    down = __uint_as_float((uint32_t)(e - 14) << 23);
}
// of all entries of the warp's accumulator tiles: one warp-wide maximum (of the bits: magnitudes order as integers)
template <int N>
__device__ __forceinline__ float frag_max(const float (&t)[N][4]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++)
        m = fmaxf(m, fmaxf(fmaxf(fabsf(t[i][0]), fabsf(t[i][1])), fmaxf(fabsf(t[i][2]), fabsf(t[i][3]))));
    return m;
}
__device__ __forceinline__ void warp_scale(float m, float& up, float& down) {
    row_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m))), up, down);
}
template <int N>
__device__ __forceinline__ void frag_scale(const float (&t)[N][4], float& up, float& down) {
    warp_scale(frag_max(t), up, down);
}
// A fragment pieces of 16 k columns of two accumulator tiles, scaled by up (an accumulator is laid out as
// an A fragment: no data moves between lanes)
template <int NP>
__device__ __forceinline__ void frag_pieces(const float (&t0)[4], const float (&t1)[4], float up,
                                            uint32_t (&a)[NP][4]) {
    uint32_t p[NP];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float* t = i < 2 ? t0 : t1;
        split_pair<NP>(t[(i & 1) * 2] * up, t[(i & 1) * 2 + 1] * up, p);
#pragma unroll
        for (int k = 0; k < NP; k++) a[k][i] = p[k];
    }
}
// acc[t] += sum over pieces of a * B for the column blocks t2 (16 columns) in [from, to): B fragments by
// load(piece, t2, regs).  Two blocks at a time keep four accumulators in turn; smaller products first.
template <int NA, int NB, int N, typename LOAD>
__device__ __forceinline__ void mma_row(float (&acc)[N][4], const uint32_t (&a)[NA][4], int from, int to,
                                        LOAD load) {
    constexpr int LIM = NA == 1 && NB == 1 ? 0 : 1;
#pragma unroll
    for (int t2 = 0; t2 < N / 2; t2 += 2) {
        if (t2 + 1 < from || t2 >= to) continue;
        uint32_t b[NB][2][4];
#pragma unroll
        for (int p = 0; p < NB; p++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                if (t2 + h >= from && t2 + h < to) load(p, t2 + h, b[p][h]);
#pragma unroll
        for (int sum = LIM; sum >= 0; sum--)
#pragma unroll
            for (int pb = 0; pb < NB; pb++)
#pragma unroll
                for (int pa = 0; pa < NA; pa++)
                    if (pa + pb == sum) {
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            if (t2 + h >= from && t2 + h < to) {
                                mma(acc[2 * (t2 + h)], a[pa], b[pb][h][0], b[pb][h][1]);
                                mma(acc[2 * (t2 + h) + 1], a[pa], b[pb][h][2], b[pb][h][3]);
                            }
                    }
    }
}

__device__ __forceinline__ float ldt(const float* p, long long i) { return p[i]; }
__device__ __forceinline__ float ldt(const __nv_bfloat16* p, long long i) { return __bfloat162float(p[i]); }
// Values as they are in memory: converted where they are used, so a load that is in flight holds nobody up.
template <typename IO> struct RawOf { using type = float; };
template <> struct RawOf<__nv_bfloat16> { using type = unsigned short; };
__device__ __forceinline__ float from_raw(float v) { return v; }
__device__ __forceinline__ float from_raw(unsigned short v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ void stt(float* p, long long i, float v) { p[i] = v; }
__device__ __forceinline__ void stt(__nv_bfloat16* p, long long i, float v) { p[i] = __float2bfloat16_rn(v); }

// first token and token count of sequence n
__device__ __forceinline__ void seq_range(const DeltaDesc& d, int n, long long& start, long long& len) {
    if (d.cu) {
        start = d.cu[n];
        len = d.cu[n + 1] - start;
    } else {
        start = (long long)n * d.T;
        len = d.T;
    }
}
// first token and tokens of a chunk; false if there is no such chunk
template <int C>
__device__ __forceinline__ bool chunk_range(const DeltaDesc& d, int chunk, long long& tok0, int& cnt) {
    int n, c;
    if (d.cu) {
        if (chunk >= d.cstart[d.nseq]) return false;
        int a = 0, b = d.nseq;   // last sequence whose first chunk is <= chunk and that is not empty
        while (b - a > 1) {
            const int m = (a + b) >> 1;
            if (d.cstart[m] <= chunk) a = m;
            else b = m;
        }
        n = a;
        c = chunk - d.cstart[n];
    } else {
        n = chunk / d.nc;
        c = chunk - n * d.nc;
    }
    long long start, len;
    seq_range(d, n, start, len);
    tok0 = start + (long long)c * C;
    cnt = (int)(len - (long long)c * C < C ? len - (long long)c * C : C);
    return true;
}

// ------------------------------------------------------------------ decays inside a chunk
// Running sums of g in 64 bits (lane holds tokens lane and lane + 32), -104 for anything below it: exp is 0 in fp32
// there, and differences of the sums stay what G needs after a reset (g = -inf) too.
__device__ __forceinline__ void running_sums(float g0, float g1, int lane, double* gam) {
    double s[2] = {g0 < -104.0f ? -104.0f : g0, g1 < -104.0f ? -104.0f : g1};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double a = __shfl_up_sync(0xffffffffu, s[0], o), b = __shfl_up_sync(0xffffffffu, s[1], o);
        if (lane >= o) {
            s[0] += a;
            s[1] += b;
        }
    }
    gam[lane] = s[0];
    gam[lane + 32] = s[1] + __shfl_sync(0xffffffffu, s[0], 31);
}
// G_ij = exp(gamma_i - gamma_j), j <= i.  Between blocks of 16 tokens it is the product of two decays that meet at
// the end of the block before i's (both at most e^0 where g <= 0, so nothing overflows on the way).
struct DecaySmem {
    double* gam;   // [C]
    float* row;    // [C]: exp(gamma_i - gamma at the end of the block before)
    float* col;    // [3][48]: exp(gamma at the end of block b - gamma_j), j <= 16 b + 15
    __device__ __forceinline__ float at(int i, int j, bool same_block, int block_i) const {
        if (same_block) return j <= i ? expf((float)(gam[i] - gam[j])) : 0.0f;
        return row[i] * col[(block_i - 1) * 48 + j];
    }
};
__device__ __forceinline__ void decay_tables(const DecaySmem& s, int tid) {   // gam is there; a barrier follows
    if (tid < kDeltaC && tid >= 16) s.row[tid] = expf((float)(s.gam[tid] - s.gam[(tid & ~15) - 1]));
    if (tid < 96) {
        const int b = tid < 16 ? 0 : tid < 48 ? 1 : 2, j = tid < 16 ? tid : tid < 48 ? tid - 16 : tid - 48;
        s.col[b * 48 + j] = expf((float)(s.gam[16 * b + 15] - s.gam[j]));
    }
}

// part[k] = A_k B_k for NK blocks of 16 of the sum, N tiles wide: all fragments are loaded before the first product and
// the products of different blocks alternate, so that neither waits for the other.  load_a(k, a), load_b(k, piece,
// t2, b).
template <int NK, int NA, int NB, int N, typename LA, typename LB>
__device__ __forceinline__ void mma_blocks(float (&part)[NK][N][4], LA load_a, LB load_b) {
    constexpr int LIM = NA == 1 && NB == 1 ? 0 : 1;
    uint32_t a[NK][NA][4], b[NK][NB][N / 2][4];
#pragma unroll
    for (int k = 0; k < NK; k++) {
        load_a(k, a[k]);
#pragma unroll
        for (int p = 0; p < NB; p++)
#pragma unroll
            for (int t = 0; t < N / 2; t++) load_b(k, p, t, b[k][p][t]);
    }
#pragma unroll
    for (int k = 0; k < NK; k++)
#pragma unroll
        for (int t = 0; t < N; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) part[k][t][e] = 0.0f;
#pragma unroll
    for (int sum = LIM; sum >= 0; sum--)
#pragma unroll
        for (int pb = 0; pb < NB; pb++)
#pragma unroll
            for (int pa = 0; pa < NA; pa++)
                if (pa + pb == sum) {
#pragma unroll
                    for (int k = 0; k < NK; k++)
#pragma unroll
                        for (int t = 0; t < N / 2; t++) {
                            mma(part[k][2 * t], a[k][pa], b[k][pb][t][0], b[k][pb][t][1]);
                            mma(part[k][2 * t + 1], a[k][pa], b[k][pb][t][2], b[k][pb][t][3]);
                        }
                }
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ------------------------------------------------------------------ chunk recurrences
// A unit is 16 columns of dv of one head.  Transposed, the state S^T [16][dk] is an m16 product's accumulator: of the
// four warps that carry the recurrence, warp w keeps quarter w of dk in registers, and owns the tokens
// 16 w .. 16 w + 15 of a chunk.  What all four need (the state, then the chunk's right-hand side, then U) goes
// through shared memory as fp16 A fragments, each warp's with a power of two of its own, so no warp waits for
// another's largest entry: the products of a block of k are summed apart and added in fp32.  Three barriers a
// chunk.  The chain of a chunk is bound by latency and by the warps' instructions, so four more warps of the unit do
// what does not carry it: the outputs, what is kept, what can be computed ahead.  A block holds NU units that
// share the staged tiles.
template <int C, int DKP, int NPK>
struct DeltaStage {
    static constexpr int KQ = NPK * C * DKP * 2;   // bytes of K (and of Q)
    static constexpr int TT = C * C * 2;           // one piece of M, T or P
    static constexpr int TOK = TOK_SIZE * 4;
    // K, Q and M or T; P and the token factors, which outputs that lag behind read a chunk later
    static constexpr int oQ = KQ, oT = 2 * KQ, FRONT = oT + 2 * TT;
    static constexpr int oTok = 2 * TT, REAR = oTok + TOK;
    static constexpr int BYTES = FRONT + REAR;

    // Bulk copies of one chunk into the stage at `front` and `rear`, M or T from `tiles`, by four threads (part
    // 0 .. 3): issuing all of them takes a warp some 500 cycles.  A copy may complete before part 0 has announced
    // the bytes.
    static __device__ __forceinline__ void load(const DeltaDesc& d, const __half* tiles, uint32_t front, uint32_t rear,
                                                uint32_t bar, int chunk, int hv, int part) {
        const int hk = hv / d.grp;
        const size_t kh = ((size_t)chunk * d.Hk + hk) * NPK * C * DKP, vh = (size_t)chunk * d.Hv + hv;
        if (part == 0) {
            mbar_expect_tx(bar, BYTES);
            bulk(rear + oTok, d.tok + vh * TOK_SIZE, TOK, bar);
            bulk(rear, d.Pt + vh * 2 * C * C, 2 * TT, bar);
        } else if (part == 1) {
            bulk(front, d.Kt + kh, KQ, bar);
        } else if (part == 2) {
            bulk(front + oQ, d.Qt + kh, KQ, bar);
        } else {
            bulk(front + oT, tiles + vh * 2 * C * C, 2 * TT, bar);
        }
    }
    static __device__ __forceinline__ void bulk(uint32_t dst, const void* src, unsigned bytes, uint32_t bar) {
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
    }
};

// A fragments in shared memory: [block][piece][lane] 16 bytes, and per block what they are times
template <int NBLK, int NP>
struct FragBuf {
    static constexpr int BYTES = NBLK * NP * 512 + 64;
    static __device__ __forceinline__ void put(unsigned char* base, int blk, int lane, const uint32_t (*a)[4],
                                               float down) {
#pragma unroll
        for (int p = 0; p < NP; p++)
            *(uint4*)(base + (blk * NP + p) * 512 + lane * 16) = make_uint4(a[p][0], a[p][1], a[p][2], a[p][3]);
        if (lane == 0) ((float*)(base + NBLK * NP * 512))[blk] = down;
    }
    static __device__ __forceinline__ void put(unsigned char* base, int blk, int lane, const float (&t)[2][4],
                                               float up, float down) {
        uint32_t a[NP][4];
        frag_pieces<NP>(t[0], t[1], up, a);
        put(base, blk, lane, a, down);
    }
    // first N of the block's pieces
    template <int N>
    static __device__ __forceinline__ void get(const unsigned char* base, int blk, int lane, uint32_t (&a)[N][4]) {
#pragma unroll
        for (int p = 0; p < N; p++) {
            const uint4 v = *(const uint4*)(base + (blk * NP + p) * 512 + lane * 16);
            a[p][0] = v.x; a[p][1] = v.y; a[p][2] = v.z; a[p][3] = v.w;
        }
    }
    static __device__ __forceinline__ float scale(const unsigned char* base, int blk) {
        return ((const float*)(base + NBLK * NP * 512))[blk];
    }
};
// A fragment pieces of one block as rows of a 16-row tile in global memory (columns col .. col + 15), W columns wide
template <int NP, int W>
__device__ __forceinline__ void put_frag(__half* base, size_t piece, int lane, int col, const uint32_t (*a)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = (lane >> 2) + 8 * (i & 1), c = col + 8 * (i >> 1) + (lane & 3) * 2;
        const uint32_t o = W == 64 ? tile_off<64>(row, c) : wide_off<16>(row, c);
#pragma unroll
        for (int k = 0; k < NP; k++) *(uint32_t*)((char*)(base + k * piece) + o) = a[k][i];
    }
}
// entries (r, c) (r, c + 1) and (r + 8, ...) of an accumulator tile, N pieces as they are
template <int W, int N = 2>
__device__ __forceinline__ void get_tile(const __half* base, size_t piece, int lane, int col, uint32_t (&v)[2][2]) {
    const int c = col + (lane & 3) * 2;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t o = W == 64 ? tile_off<64>((lane >> 2) + 8 * h, c) : wide_off<16>((lane >> 2) + 8 * h, c);
#pragma unroll
        for (int k = 0; k < N; k++) v[h][k] = *(const uint32_t*)((const char*)(base + k * piece) + o);
    }
}
// x, y of a pair of pieces
__device__ __forceinline__ float2 join(uint32_t hi, uint32_t lo) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    return make_float2(a.x + b.x, a.y + b.y);
}
template <int N>
__device__ __forceinline__ void zero(float (&t)[N][4]) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) t[i][e] = 0.0f;
}
// acc += f part
template <int N>
__device__ __forceinline__ void add_scaled(float (&acc)[N][4], const float (&part)[N][4], float f) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[i][e] = fmaf(part[i][e], f, acc[i][e]);
}
// acc += f part if `on` (0 or ~0).  The triangular products run over all blocks without a branch, so that they overlap;
// those outside the triangle, whose factors hold anything, are masked out here.
template <int N>
__device__ __forceinline__ void add_masked(float (&acc)[N][4], const float (&part)[N][4], float f, uint32_t on) {
    f = __uint_as_float(__float_as_uint(f) & on);
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            acc[i][e] = fmaf(__uint_as_float(__float_as_uint(part[i][e]) & on), f, acc[i][e]);
}
// barriers of unit g: its chain warps, its side warps, all of them
__device__ __forceinline__ void chain_bar(int g) { asm volatile("bar.sync %0, 128;" ::"r"(3 * g + 1) : "memory"); }
__device__ __forceinline__ void side_bar(int g) { asm volatile("bar.sync %0, 128;" ::"r"(3 * g + 2) : "memory"); }
__device__ __forceinline__ void unit_bar(int g) { asm volatile("bar.sync %0, 256;" ::"r"(3 * g + 3) : "memory"); }
// A warp's 16 tokens x 16 columns of v or dO as accumulator tiles [16 columns][2 x 8 tokens].  bf16 rows on 16-byte
// boundaries (vec): one 16-byte load per lane, held as it is until the tiles are needed, then transposed by ldmatrix
// through 512 bytes of the warp's own; else entry by entry.
template <typename IO>
struct TokenTile {
    using RT = typename RawOf<IO>::type;
    uint4 w;
    RT e[2][4];
    __device__ __forceinline__ void load(const void* base, long long tok, long long ld, long long at, int cols, int n,
                                         int lane, bool vec) {
        if (sizeof(IO) == 2 && vec) {
            const int t = lane >> 1, c = (lane & 1) * 8;
            w = t < n && c < cols ? *(const uint4*)((const RT*)base + (tok + t) * ld + at + c) : make_uint4(0, 0, 0, 0);
            return;
        }
        const int r = lane >> 2, c2 = (lane & 3) * 2;
        const RT* p = (const RT*)base + tok * ld + at + r;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int i = t * 8 + c2 + (k & 1);
                e[t][k] = i < n && r + (k >> 1) * 8 < cols ? p[(long long)i * ld + (k >> 1) * 8] : RT(0);
            }
    }
    __device__ __forceinline__ void tiles(float (&x)[2][4], unsigned char* scratch, int lane, bool vec) const {
        if (sizeof(IO) == 2 && vec) {
            *(uint4*)(scratch + lane * 16) = w;   // [token][16 columns]
            __syncwarp();
            uint32_t f[4];   // columns 0-7, 8-15 of tokens 0-7, then of 8-15
            ldm4t(f, (uint32_t)__cvta_generic_to_shared(scratch) + ((lane & 7) + (lane >> 4) * 8) * 32 + ((lane >> 3) & 1) * 16);
            __syncwarp();
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    x[t][h * 2] = __uint_as_float(f[t * 2 + h] << 16);
                    x[t][h * 2 + 1] = __uint_as_float(f[t * 2 + h] & 0xffff0000u);
                }
            return;
        }
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int k = 0; k < 4; k++) x[t][k] = from_raw(e[t][k]);
    }
};
// accumulator tiles through shared memory, [tile][lane] 16 bytes
template <int N>
__device__ __forceinline__ void put_acc(unsigned char* base, int tile, int lane, const float (&t)[N][4]) {
#pragma unroll
    for (int i = 0; i < N; i++)
        *(float4*)(base + (tile + i) * 512 + lane * 16) = make_float4(t[i][0], t[i][1], t[i][2], t[i][3]);
}
template <int N>
__device__ __forceinline__ void get_acc(const unsigned char* base, int tile, int lane, float (&t)[N][4]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float4 v = *(const float4*)(base + (tile + i) * 512 + lane * 16);
        t[i][0] = v.x; t[i][1] = v.y; t[i][2] = v.z; t[i][3] = v.w;
    }
}

int delta_sms();
// Units per block.  One gives the shorter chain, two more units per SM.  Sequences of one length: two above one unit
// per SM (16384 tokens, 8 heads of 64, bf16, forward with keep / backward in us, one and two: 128 units 192 / 293 and 262 /
// 348, 256 units 191 / 295 and 166 / 253).  Packed sequences are of unknown lengths, and the longest's chain is what
// counts until there are several times as many units as SMs (random lengths, heads of 64: 512 units 190 / 300 and 251 / 342,
// 1024 units 204 / 311 and 183 / 275; heads of 128: 512 units 390 / 702 and 369 / 721, 1024 units 393 / 707 and 339 / 688).
inline int delta_units(const DeltaDesc& d) {
    const long long all = (long long)d.nseq * d.Hv * d.units;
    return d.units > 1 && all > (d.cu ? 4 : 1) * delta_sms() ? 2 : 1;
}

cudaError_t delta_chain_fwd(const DeltaDesc& d, int DKP, bool bf16, bool keep, cudaStream_t st);
cudaError_t delta_chain_bwd(const DeltaDesc& d, int DKP, bool bf16, cudaStream_t st);
cudaError_t delta_grads(const DeltaDesc& d, int DKP, bool bf16, cudaStream_t st);

}  // namespace kmb
