// layernorm.cu -- layer norm with its residual, forward and backward
// (include/kmamba_norm.h).
//
// Both directions are bound by HBM: the forward moves x, residual, s and y, the
// backward s, dy, dtotal and dx, once each.  A row is read once into registers
// and everything about it is computed there: the mean, then the centred square
// sum (two passes over registers, so there is no cancellation), then the output.
// Rows up to 512 entries belong to one warp (no block barrier, the 8 warps of a
// block run on independent rows), longer rows to a block of 8 or 16 entries per
// thread, so that enough warps fit an SM to keep its loads in flight.
//
// The weight's gradient is a sum over all rows: each thread keeps its columns in
// registers over all of its rows, a block adds its warps in order, and a second
// launch adds the blocks' partial sums in order.  No atomics: the result does
// not depend on scheduling.
//
// Measured at 131072 x 512 bf16 with residual: forward 82 us (537 MB, 6.5 TB/s: a
// copy's rate), backward with the weight's gradient 121 us (4.4 TB/s; its 500
// instructions a row and warp fill half of the issue slots); 10007 x 1001 fp32: 24 and
// 42 us, rows of blocks of 128 threads that wait for two block sums each.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include "../../include/kmamba_norm.h"
#include "kmb_launch.cuh"

namespace kmb {
int set_error(const char* msg);
int set_cuda_error(const char* where, cudaError_t e);
void clear_error();

namespace {

constexpr int LN_WARP_D = 512;    // longest row of the warp kernels
constexpr int LN_BLOCK8_D = 8192; // longest row of blocks with 8 entries per thread
constexpr int LN_BWD_BLOCKS = 2;   // blocks of the warp kernels per SM in the backward
constexpr int LN_WARPS = 8;       // rows in flight per block there

struct LnDesc {
    long long rows;
    int D;
    float eps;
    const void *x, *res, *dy, *dtot;
    void *tot, *y, *dx;
    const float *w, *b;
    float *mean, *rstd;
    long long ld_x, ld_res, ld_tot, ld_y, ld_dy, ld_dtot, ld_dx;
    float* part;        // [blocks][2][D] partial dw, db
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

// VEC elements of T as they are in memory (bf16 pairs stay packed: one register)
template <typename T, int VEC> struct Raw {
    T e[VEC];
    __device__ __forceinline__ float get(int j) const { return to_f(e[j]); }
    __device__ __forceinline__ void set(const float (&v)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; j++) from_f(v[j], e[j]);
    }
};
template <> struct __align__(16) Raw<float, 4> {
    float e[4];
    __device__ __forceinline__ float get(int j) const { return e[j]; }
    __device__ __forceinline__ void set(const float (&v)[4]) {
#pragma unroll
        for (int j = 0; j < 4; j++) e[j] = v[j];
    }
};
template <> struct __align__(16) Raw<__nv_bfloat16, 8> {
    uint32_t w[4];
    __device__ __forceinline__ float get(int j) const {
        return __uint_as_float((j & 1) ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
};

template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> ld_raw(const T* p) {
    return *reinterpret_cast<const Raw<T, VEC>*>(p);
}
template <int VEC>
__device__ __forceinline__ void ld_f(const float* p, float (&v)[VEC]) {
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 t = *reinterpret_cast<const float4*>(p + i);
            v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = p[i];
    }
}

// VEC columns from `col`, whose address is aligned; columns outside [0, D) read as 0 and are not written
template <typename T, int VEC, bool ODD>
__device__ __forceinline__ Raw<T, VEC> ld_cols(const T* row, int col, int D) {
    if (!ODD || (col >= 0 && col + VEC <= D)) return ld_raw<T, VEC>(row + col);
    Raw<T, VEC> r;
    float v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) v[j] = col + j >= 0 && col + j < D ? to_f(row[col + j]) : 0.0f;
    r.set(v);
    return r;
}
template <typename T, int VEC, bool ODD>
__device__ __forceinline__ void st_cols(T* row, int col, int D, const Raw<T, VEC>& r) {
    if (!ODD || (col >= 0 && col + VEC <= D)) {
        *reinterpret_cast<Raw<T, VEC>*>(row + col) = r;
        return;
    }
#pragma unroll
    for (int j = 0; j < VEC; j++)
        if (col + j >= 0 && col + j < D) from_f(r.get(j), row[col + j]);
}
template <int VEC, bool ODD>
__device__ __forceinline__ void ld_w(const float* p, int col, int D, float (&v)[VEC]) {
    if constexpr (!ODD) {
        ld_f<VEC>(p + col, v);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) v[j] = col + j >= 0 && col + j < D ? p[col + j] : 0.0f;
    }
}
// Entries between a 16-byte boundary and the start of a row: its chunks start that many columns early.  The rows of a
// thread are a multiple of 8 apart, so it is the same for all of them.
template <typename T, bool ODD>
__device__ __forceinline__ int early(const T* row) {
    return ODD ? (int)(((uintptr_t)row & 15) / sizeof(T)) : 0;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// sum over the threads of a row: a warp, or the whole block (same order every time)
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float v, float* sh) {
    v = warp_sum(v);
    if constexpr (BLOCK) {
        const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sh[warp] = v;
        __syncthreads();
        v = (threadIdx.x & 31) < nw ? sh[threadIdx.x & 31] : 0.0f;
        v = warp_sum(v);
    }
    return v;
}

// NCH chunks of VEC consecutive columns per thread, chunks TPR * VEC columns apart.
template <typename T, int VEC, int NCH, bool BLOCK, bool ODD>
__global__ void __launch_bounds__(BLOCK ? 1024 : 32 * LN_WARPS)
ln_fwd_kernel(const LnDesc d) {
    __shared__ float sh[32];
    const int lane = BLOCK ? threadIdx.x : (threadIdx.x & 31);
    const int tpr = BLOCK ? blockDim.x : 32;
    const long long row = BLOCK ? (long long)blockIdx.x
                                : (long long)blockIdx.x * LN_WARPS + (threadIdx.x >> 5);
    if (row >= d.rows) return;   // warps of their own, or the whole block
    const T* x = (const T*)d.x + row * d.ld_x;
    const T* r = (const T*)d.res + row * d.ld_res;
    const int sft = early<T, ODD>(x);
    const bool has_res = d.res != nullptr;
    const auto at = [&](int i) { return (i * tpr + lane) * VEC - sft; };
    const auto in = [&](int c) { return ODD ? c >= 0 && c < d.D : true; };   // of a chunk that starts before D
    float v[NCH][VEC];
    {
        Raw<T, VEC> a[NCH], c[NCH];
#pragma unroll
        for (int i = 0; i < NCH; i++)
            if (at(i) < d.D) a[i] = ld_cols<T, VEC, ODD>(x, at(i), d.D);
        if (has_res) {
#pragma unroll
            for (int i = 0; i < NCH; i++)
                if (at(i) < d.D) c[i] = ld_cols<T, VEC, ODD>(r, at(i), d.D);
        }
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            if (at(i) < d.D) {
                if (has_res) {
                    float t[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; j++) t[j] = a[i].get(j) + c[i].get(j);
                    a[i].set(t);
                    if (d.tot) st_cols<T, VEC, ODD>((T*)d.tot + row * d.ld_tot, at(i), d.D, a[i]);
                }
#pragma unroll
                for (int j = 0; j < VEC; j++) v[i][j] = a[i].get(j);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; j++) v[i][j] = 0.0f;
            }
        }
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NCH; i++)
#pragma unroll
        for (int j = 0; j < VEC; j++) s += v[i][j];
    const float mean = row_sum<BLOCK>(s, sh) / (float)d.D;
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < NCH; i++)
        if (at(i) < d.D) {
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                v[i][j] = in(at(i) + j) ? v[i][j] - mean : 0.0f;
                q = fmaf(v[i][j], v[i][j], q);
            }
        }
    const float rstd = 1.0f / sqrtf(row_sum<BLOCK>(q, sh) / (float)d.D + d.eps);
    if (d.mean && lane == 0) {
        d.mean[row] = mean;
        d.rstd[row] = rstd;
    }
    T* y = (T*)d.y + row * d.ld_y;
#pragma unroll
    for (int i = 0; i < NCH; i++) {
        if (at(i) < d.D) {
            float w[VEC], b[VEC];
            float y8[VEC];
            Raw<T, VEC> o;
            if (d.w) ld_w<VEC, ODD>(d.w, at(i), d.D, w);
            if (d.b) ld_w<VEC, ODD>(d.b, at(i), d.D, b);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const float h = v[i][j] * rstd;
                y8[j] = fmaf(h, d.w ? w[j] : 1.0f, d.b ? b[j] : 0.0f);
            }
            o.set(y8);
            st_cols<T, VEC, ODD>(y, at(i), d.D, o);
        }
    }
}

// Backward.  Blocks walk rows with the grid's stride; the normalised entries are computed twice.  Where a warp's rows
// are aligned (PRE) they come through a ring of shared memory filled by cp.async, two rows ahead (each lane reads
// what it copied itself, so the warp never waits for another): keeping two rows in registers instead held 128
// of them and took 135 us at 131072 x 512 bf16, against 104; three blocks per SM spilled (179 in that form).  Elsewhere a row stays in registers as it is in memory.
template <typename T, int VEC, int NCH, bool BLOCK>
struct LnBwd {
    static constexpr int E = NCH * VEC;
    static constexpr int MIN_BLOCKS = BLOCK ? 1 : LN_BWD_BLOCKS;
    static constexpr int SLOT = NCH * 512;                        // bytes of one tensor's row (32 lanes x 16 x NCH)
    static constexpr int DEPTH = SLOT <= 1024 ? 3 : 2;
    static constexpr int RING = LN_WARPS * DEPTH * 3 * SLOT;
};
template <typename T, int VEC, int NCH, bool BLOCK, bool ODD>
__global__ void __launch_bounds__(BLOCK ? 1024 : 32 * LN_WARPS, (LnBwd<T, VEC, NCH, BLOCK>::MIN_BLOCKS))
ln_bwd_kernel(const LnDesc d) {
    using B = LnBwd<T, VEC, NCH, BLOCK>;
    constexpr bool PRE = !BLOCK && !ODD && VEC > 1;
    extern __shared__ __align__(16) float dynsh[];   // warp rows: [2][D] to add the warps in, over the ring
    __shared__ float sh[32];
    const int lane = BLOCK ? threadIdx.x : (threadIdx.x & 31);
    const int warp = threadIdx.x >> 5;
    const int tpr = BLOCK ? blockDim.x : 32;
    const long long first = BLOCK ? (long long)blockIdx.x : (long long)blockIdx.x * LN_WARPS + warp;
    const long long step = BLOCK ? (long long)gridDim.x : (long long)gridDim.x * LN_WARPS;
    // (a thread of a row that does not exist reads nothing)
    const int sft = early<T, ODD>((const T*)d.x + first * d.ld_x);
    const auto at = [&](int i) { return (i * tpr + lane) * VEC - sft; };
    const auto in = [&](int c) { return ODD ? c >= 0 && c < d.D : true; };
    float aw[NCH][VEC], ab[NCH][VEC];
    pdl_release();
#pragma unroll
    for (int i = 0; i < NCH; i++)
#pragma unroll
        for (int j = 0; j < VEC; j++) aw[i][j] = ab[i][j] = 0.0f;
    struct Row {
        Raw<T, VEC> s[NCH], dy[NCH], t[NCH];
        float mean, rstd;
    };
    const bool has_t = d.dtot != nullptr;
    const float inv_d = 1.0f / (float)d.D;
    auto load = [&](long long row, Row& r) {
        const T* s = (const T*)d.x + row * d.ld_x;
        const T* dy = (const T*)d.dy + row * d.ld_dy;
        const T* t = (const T*)d.dtot + row * d.ld_dtot;
#pragma unroll
        for (int i = 0; i < NCH; i++)
            if (at(i) < d.D) {
                r.s[i] = ld_cols<T, VEC, ODD>(s, at(i), d.D);
                r.dy[i] = ld_cols<T, VEC, ODD>(dy, at(i), d.D);
                if (has_t) r.t[i] = ld_cols<T, VEC, ODD>(t, at(i), d.D);
            }
        r.mean = d.mean[row];
        r.rstd = d.rstd[row];
    };
    // get(k, i): 16-byte pieces of s, dy, dtotal (k = 0, 1, 2)
    auto work = [&](long long row, float mean, float rstd, auto get) {
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            const int col = at(i);
            if (col < d.D) {
                float w[VEC];
                if (d.w) ld_w<VEC, ODD>(d.w, col, d.D, w);
                const Raw<T, VEC> rs = get(0, i), ry = get(1, i);
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const float xh = (rs.get(j) - mean) * rstd;
                    const float dy = ry.get(j);   // 0 outside the row
                    aw[i][j] = fmaf(dy, xh, aw[i][j]);
                    ab[i][j] += dy;
                    const float g = d.w ? __fmul_rn(dy, w[j]) : dy;
                    s1 += g;
                    s2 = fmaf(g, xh, s2);
                }
            }
        }
        s1 = row_sum<BLOCK>(s1, sh) * inv_d;
        s2 = row_sum<BLOCK>(s2, sh) * inv_d;
        if (!d.dx) return;
        T* dx = (T*)d.dx + row * d.ld_dx;
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            const int col = at(i);
            if (col < d.D) {
                float w[VEC], o8[VEC];
                if (d.w) ld_w<VEC, ODD>(d.w, col, d.D, w);
                const Raw<T, VEC> rs = get(0, i), ry = get(1, i);
                Raw<T, VEC> rt, o;
                if (has_t) rt = get(2, i);
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const float xh = (rs.get(j) - mean) * rstd;
                    const float dy = ry.get(j);
                    // the product is rounded as in the sums: two columns (or one) cancel to what eps leaves
                    o8[j] = rstd * ((d.w ? __fmul_rn(dy, w[j]) : dy) - s1 - xh * s2);
                    if (has_t) o8[j] += rt.get(j);
                }
                o.set(o8);
                st_cols<T, VEC, ODD>(dx, col, d.D, o);
            }
        }
    };
    if constexpr (PRE) {
        // dx may be dy or dtotal: the rows ahead belong to this warp alone, nobody writes them before they are copied
        unsigned char* ring = (unsigned char*)dynsh + warp * (B::DEPTH * 3 * B::SLOT) + lane * 16;
        const uint32_t ra = (uint32_t)__cvta_generic_to_shared(ring);
        const auto copy = [&](long long k) {
            const long long row = first + k * step;
            if (row < d.rows) {
                const T* src[3] = {(const T*)d.x + row * d.ld_x, (const T*)d.dy + row * d.ld_dy,
                                   (const T*)d.dtot + row * d.ld_dtot};
                const uint32_t dst = ra + (uint32_t)(k % B::DEPTH) * (3 * B::SLOT);
#pragma unroll
                for (int i = 0; i < NCH; i++)
                    if (at(i) < d.D) {
#pragma unroll
                        for (int t = 0; t < 3; t++)
                            if (t < 2 || has_t)
                                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                                             ::"r"(dst + t * B::SLOT + i * 512), "l"(src[t] + at(i)) : "memory");
                    }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int k = 0; k < B::DEPTH - 1; k++) copy(k);
        float mS = 0.0f, rS = 0.0f;   // statistics of 32 rows, one per lane
        long long k = 0;
        for (long long row = first; row < d.rows; row += step, k++) {
            copy(k + B::DEPTH - 1);
            if ((k & 31) == 0) {
                const long long mine = row + lane * step;
                mS = mine < d.rows ? d.mean[mine] : 0.0f;
                rS = mine < d.rows ? d.rstd[mine] : 0.0f;
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(B::DEPTH - 1) : "memory");
            const unsigned char* slot = ring + (k % B::DEPTH) * (3 * B::SLOT);
            work(row, __shfl_sync(0xffffffffu, mS, k & 31), __shfl_sync(0xffffffffu, rS, k & 31),
                 [&](int t, int i) { return *(const Raw<T, VEC>*)(slot + t * B::SLOT + i * 512); });
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
        for (long long row = first; row < d.rows; row += step) {
            Row a;
            load(row, a);
            work(row, a.mean, a.rstd, [&](int t, int i) { return t == 0 ? a.s[i] : t == 1 ? a.dy[i] : a.t[i]; });
        }
    }
    if (!d.part) return;
    float* part = d.part + (size_t)blockIdx.x * 2 * d.D;
    if constexpr (BLOCK) {
#pragma unroll
        for (int i = 0; i < NCH; i++)
            if (at(i) < d.D) {
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    if (in(at(i) + j)) {
                        part[at(i) + j] = aw[i][j];
                        part[d.D + at(i) + j] = ab[i][j];
                    }
            }
    } else {
        __syncthreads();                       // the ring is read
        for (int k = 0; k < LN_WARPS; k++) {   // the warps add in order
            if (warp == k) {
#pragma unroll
                for (int i = 0; i < NCH; i++) {
                    const int col = at(i);
                    if (col < d.D) {
#pragma unroll
                        for (int j = 0; j < VEC; j++)
                            if (in(col + j)) {
                                dynsh[col + j] = k ? dynsh[col + j] + aw[i][j] : aw[i][j];
                                dynsh[d.D + col + j] = k ? dynsh[d.D + col + j] + ab[i][j] : ab[i][j];
                            }
                    }
                }
            }
            __syncthreads();
        }
        for (int i = threadIdx.x; i < 2 * d.D; i += blockDim.x) part[i] = dynsh[i];
    }
}

// dw[c], db[c] (+)= sum over the blocks' partial sums, in a fixed order: 32 columns per block, 32 interleaved runs of
// the partial sums, four loads of each in flight, the runs added in order.
__global__ void __launch_bounds__(1024) ln_reduce_kernel(const float* part, int nb, int D, float* dw, float* db,
                                                         int accumulate) {
    __shared__ float sh[32][33];
    pdl_wait();
    const int c = blockIdx.x * 32 + threadIdx.x, g = threadIdx.y;
    float v = 0.0f;
    if (c < 2 * D) {
        int b = g;
        for (; b + 96 < nb; b += 128) {
            const float* p = part + (size_t)b * 2 * D + c;
            const size_t s = (size_t)64 * D;
            v += (p[0] + p[s]) + (p[2 * s] + p[3 * s]);
        }
        for (; b < nb; b += 32) v += part[(size_t)b * 2 * D + c];
    }
    sh[g][threadIdx.x] = v;
    __syncthreads();
    if (g == 0 && c < 2 * D) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; k++) s += sh[k][threadIdx.x];
        float* o = c < D ? dw : db;
        const int i = c < D ? c : c - D;
        if (o) o[i] = accumulate ? o[i] + s : s;
    }
}

int sm_count() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// How rows are read: 0 = in 16-byte pieces, every row of every tensor starts on 16 bytes; 1 = in 16-byte pieces
// that start before the row, all tensors' rows being off the boundary by the same amount; 2 = by single entries.
template <typename T>
int row_form(const LnDesc& d, bool bwd) {
    const int V = 16 / (int)sizeof(T);
    const void* p[5] = {d.x, bwd ? d.dy : d.res, bwd ? d.dtot : d.tot, bwd ? d.dx : d.y, nullptr};
    const long long ld[5] = {d.ld_x, bwd ? d.ld_dy : d.ld_res, bwd ? d.ld_dtot : d.ld_tot, bwd ? d.ld_dx : d.ld_y, 0};
    bool even = d.D % V == 0 && aligned16(d.w) && (bwd || aligned16(d.b)), alike = true;
    for (int i = 0; i < 4; i++) {
        if (!p[i]) continue;
        even = even && aligned16(p[i]) && ld[i] % V == 0;
        alike = alike && (((uintptr_t)p[i] ^ (uintptr_t)d.x) & 15) == 0 && (ld[i] - d.ld_x) % V == 0 &&
                ((uintptr_t)p[i] % sizeof(T)) == 0;
    }
    return even ? 0 : alike ? 1 : 2;
}

int block_entries(int D) { return D <= LN_BLOCK8_D ? 8 : 16; }
int block_threads(int D) {
    const int t = ((D + block_entries(D) - 1) / block_entries(D) + 31) & ~31;
    return t < 64 ? 64 : t > 1024 ? 1024 : t;
}
// Blocks of the backward: enough to fill the device once (the partial sums of dw and db grow with them), a multiple
// of 8 where they walk several rows.  span: columns that a row's chunks cover.
int bwd_blocks(long long rows, int span) {
    long long per_sm = LN_BWD_BLOCKS, want = (rows + LN_WARPS - 1) / LN_WARPS;
    if (span > LN_WARP_D) {
        per_sm = 1024 / block_threads(span);
        per_sm = per_sm < 1 ? 1 : per_sm;
        want = rows;
    }
    const long long cap = (per_sm * sm_count() + 7) & ~7LL;
    return (int)(want < cap ? (want > 0 ? want : 1) : cap);
}
template <typename T>
int span_of(const LnDesc& d, int form) { return d.D + (form == 1 ? 16 / (int)sizeof(T) - 1 : 0); }
template <typename T, bool BWD>
int form_of(const LnDesc& d) {
    const int form = row_form<T>(d, BWD);
    // the longest rows would need more threads than a block has
    return form == 1 && span_of<T>(d, 1) > KMB_NORM_MAX_D ? 2 : form;
}

template <typename T, int VEC, int NCH, bool BLOCK, bool ODD>
cudaError_t fwd_go(const LnDesc& d, cudaStream_t st) {
    const long long blocks = BLOCK ? d.rows : (d.rows + LN_WARPS - 1) / LN_WARPS;
    const int threads = BLOCK ? block_threads(d.D + (ODD ? VEC - 1 : 0)) : 32 * LN_WARPS;
    ln_fwd_kernel<T, VEC, NCH, BLOCK, ODD><<<(unsigned)blocks, threads, 0, st>>>(d);
    return cudaGetLastError();
}
template <typename T, int VEC, int NCH, bool BLOCK, bool ODD>
cudaError_t bwd_go(const LnDesc& d, cudaStream_t st) {
    using B = LnBwd<T, VEC, NCH, BLOCK>;
    const size_t ring = !BLOCK && !ODD && VEC > 1 ? B::RING : 0, add = (size_t)2 * d.D * sizeof(float);
    const size_t sm = BLOCK ? 0 : ring > add ? ring : add;
    if (sm > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(ln_bwd_kernel<T, VEC, NCH, BLOCK, ODD>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm);
        if (e != cudaSuccess) return e;
    }
    const int threads = BLOCK ? block_threads(d.D + (ODD ? VEC - 1 : 0)) : 32 * LN_WARPS;
    ln_bwd_kernel<T, VEC, NCH, BLOCK, ODD><<<bwd_blocks(d.rows, d.D + (ODD ? VEC - 1 : 0)), threads, sm, st>>>(d);
    return cudaGetLastError();
}

template <typename T, int VEC, bool BWD, bool ODD>
cudaError_t pick(const LnDesc& d, cudaStream_t st) {
    const int D = d.D + (ODD ? VEC - 1 : 0);   // columns that the chunks may have to span
    if (D > LN_WARP_D) {
        if (block_entries(D) == 16) {
            if constexpr (BWD) return bwd_go<T, VEC, 16 / VEC, true, ODD>(d, st);
            else return fwd_go<T, VEC, 16 / VEC, true, ODD>(d, st);
        }
        if constexpr (BWD) return bwd_go<T, VEC, 8 / VEC, true, ODD>(d, st);
        else return fwd_go<T, VEC, 8 / VEC, true, ODD>(d, st);
    }
    // entries per lane: 8 or 16
#define KMB_LN_GO(E)                                                       \
    {                                                                      \
        if constexpr (BWD) return bwd_go<T, VEC, E / VEC, false, ODD>(d, st); \
        else return fwd_go<T, VEC, E / VEC, false, ODD>(d, st);            \
    }
    if (D <= 256) KMB_LN_GO(8)
    KMB_LN_GO(16)
#undef KMB_LN_GO
}
template <typename T, bool BWD>
cudaError_t dispatch_t(const LnDesc& d, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const int form = form_of<T, BWD>(d);
    if (form == 0) return pick<T, V, BWD, false>(d, st);
    if (form == 1) return pick<T, V, BWD, true>(d, st);
    return pick<T, 1, BWD, false>(d, st);
}
template <bool BWD>
cudaError_t dispatch(const LnDesc& d, int dtype, cudaStream_t st) {
    return dtype == KMB_DTYPE_BF16 ? dispatch_t<__nv_bfloat16, BWD>(d, st) : dispatch_t<float, BWD>(d, st);
}

const char* check(const KMBNormParams* p) {
    if (!p) return "layernorm: null parameters";
    if (p->rows < 0 || p->D < 1 || p->D > KMB_NORM_MAX_D) return "layernorm: rows must be >= 0 and D in 1 .. 16384";
    if (p->rows > 0x7fffffffLL) return "layernorm: at most 2^31 - 1 rows";
    if (p->dtype != KMB_DTYPE_F32 && p->dtype != KMB_DTYPE_BF16) return "layernorm: unknown dtype";
    if (!(p->eps >= 0.0f)) return "layernorm: eps must be >= 0";
    if ((p->mean == nullptr) != (p->rstd == nullptr)) return "layernorm: mean and rstd go together";
    const long ld[] = {p->ld_x, p->ld_residual, p->ld_total, p->ld_y};
    for (long l : ld)
        if (l != 0 && l < p->D) return "layernorm: a row stride is shorter than D";
    return nullptr;
}
// whether one of the pointers is off its element's boundary (an access there is an error of the device)
bool off(size_t size, std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if ((uintptr_t)p % size) return true;
    return false;
}
constexpr const char* kOff = "layernorm: a tensor is not aligned to its elements";
size_t elem(const KMBNormParams* p) { return p->dtype == KMB_DTYPE_BF16 ? 2 : 4; }
bool off(const KMBNormParams* p) {
    return off(elem(p), {p->x, p->residual, p->total, p->y}) || off(4, {p->w, p->b, p->mean, p->rstd});
}
long long or_d(long ld, long D) { return ld ? ld : D; }

}  // namespace
}  // namespace kmb

using namespace kmb;

extern "C" {

int kmb_layernorm_forward(const KMBNormParams* p, void* stream) {
    clear_error();
    if (const char* m = check(p)) return set_error(m);
    if (p->rows == 0) return 0;
    if (!p->x || !p->y) return set_error("layernorm: x and y are required");
    if (p->total && !p->residual) return set_error("layernorm: total without a residual");
    if (off(p)) return set_error(kOff);
    LnDesc d{};
    d.rows = p->rows; d.D = (int)p->D; d.eps = p->eps;
    d.x = p->x; d.res = p->residual; d.tot = p->total; d.y = p->y; d.w = p->w; d.b = p->b;
    d.mean = p->mean; d.rstd = p->rstd;
    d.ld_x = or_d(p->ld_x, p->D); d.ld_res = or_d(p->ld_residual, p->D); d.ld_tot = or_d(p->ld_total, p->D);
    d.ld_y = or_d(p->ld_y, p->D);
    cudaError_t e = dispatch<false>(d, p->dtype, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : set_cuda_error("kmb_layernorm_forward", e);
}

size_t kmb_layernorm_workspace_floats(const KMBNormParams* p) {
    if (check(p)) return 0;
    // the larger of what rows on and off 16-byte boundaries take
    const int a = bwd_blocks(p->rows, (int)p->D), b = bwd_blocks(p->rows, (int)p->D + 7);
    return (size_t)(a > b ? a : b) * 2 * p->D;
}

int kmb_layernorm_backward(const KMBNormParams* p, const KMBNormGrads* g, float* ws, void* stream) {
    clear_error();
    if (const char* m = check(p)) return set_error(m);
    if (!g) return set_error("layernorm backward: null gradients");
    const long ld[] = {g->ld_dy, g->ld_dtotal, g->ld_dx};
    for (long l : ld)
        if (l != 0 && l < p->D) return set_error("layernorm backward: a row stride is shorter than D");
    const bool wgrad = g->dw || g->db;
    cudaStream_t st = (cudaStream_t)stream;
    if (p->rows == 0) {   // no rows: the sums over them are zero
        if (!g->accumulate) {
            cudaError_t e = cudaSuccess;
            if (g->dw) e = cudaMemsetAsync(g->dw, 0, p->D * sizeof(float), st);
            if (e == cudaSuccess && g->db) e = cudaMemsetAsync(g->db, 0, p->D * sizeof(float), st);
            if (e != cudaSuccess) return set_cuda_error("kmb_layernorm_backward", e);
        }
        return 0;
    }
    const void* s = p->residual ? p->total : p->x;
    if (!s) return set_error("layernorm backward: the normalised input (total, or x without a residual) is required");
    if (!p->mean || !g->dy) return set_error("layernorm backward: mean, rstd and dy are required");
    if (wgrad && !ws) return set_error("layernorm backward: dw and db need the workspace");
    if (off(p) || off(elem(p), {g->dy, g->dtotal, g->dx}) || off(4, {g->dw, g->db, ws})) return set_error(kOff);
    LnDesc d{};
    d.rows = p->rows; d.D = (int)p->D; d.eps = p->eps;
    d.x = s; d.ld_x = p->residual ? or_d(p->ld_total, p->D) : or_d(p->ld_x, p->D);
    d.dy = g->dy; d.dtot = g->dtotal; d.dx = g->dx; d.w = p->w; d.mean = p->mean; d.rstd = p->rstd;
    d.ld_dy = or_d(g->ld_dy, p->D); d.ld_dtot = or_d(g->ld_dtotal, p->D); d.ld_dx = or_d(g->ld_dx, p->D);
    d.part = wgrad ? ws : nullptr;
    cudaError_t e = dispatch<true>(d, p->dtype, st);
    if (e == cudaSuccess && wgrad) {
        const int span = p->dtype == KMB_DTYPE_BF16 ? span_of<__nv_bfloat16>(d, form_of<__nv_bfloat16, true>(d))
                                                    : span_of<float>(d, form_of<float, true>(d));
        e = launch(ln_reduce_kernel, dim3((unsigned)((2 * p->D + 31) / 32)), dim3(32, 32), 0, st, true, ws,
                   bwd_blocks(p->rows, span), (int)p->D, g->dw, g->db, g->accumulate);
    }
    return e == cudaSuccess ? 0 : set_cuda_error("kmb_layernorm_backward", e);
}

}  // extern "C"
