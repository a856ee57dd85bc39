// layernorm.cu -- layer norm with its residual, forward and backward
// (include/kmamba_norm.h).
//
// Both directions are bound by HBM: the forward moves x, residual, s and y, the
// backward s, dy, dtotal and dx, once each.  A row is read once into registers
// and everything about it is computed there: the mean, then the centred square
// sum (two passes over registers, so there is no cancellation), then the output.
// Rows up to 1024 entries belong to one warp (no block barrier, the 8 warps of a
// block run on independent rows); longer rows belong to a block.
//
// The weight's gradient is a sum over all rows: each warp keeps its lanes'
// columns in registers over all of its rows (a block with long rows keeps them
// in shared memory, every column owned by one thread), the block adds its warps
// in order, and a second launch adds the blocks' partial sums in order.  No
// atomics: the result does not depend on scheduling.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cmath>
#include <cstdint>
#include "../../include/kmamba_norm.h"

namespace kmb {
int set_error(const char* msg);
int set_cuda_error(const char* where, cudaError_t e);
void clear_error();

namespace {

constexpr int LN_WARP_D = 1024;   // longest row of the warp kernels
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

// VEC elements of T as they are in memory
template <typename T, int VEC> struct Raw { T e[VEC]; };
template <> struct __align__(16) Raw<float, 4> { float e[4]; };
template <> struct __align__(16) Raw<__nv_bfloat16, 8> { __nv_bfloat16 e[8]; };
template <> struct __align__(4) Raw<__nv_bfloat16, 2> { __nv_bfloat16 e[2]; };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

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
template <typename T, int VEC, int NCH, bool BLOCK>
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
    const bool has_res = d.res != nullptr;
    float v[NCH][VEC];
    {
        Raw<T, VEC> a[NCH], c[NCH];
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            const int col = (i * tpr + lane) * VEC;
            if (col < d.D) a[i] = ld_raw<T, VEC>(x + col);
        }
        if (has_res) {
#pragma unroll
            for (int i = 0; i < NCH; i++) {
                const int col = (i * tpr + lane) * VEC;
                if (col < d.D) c[i] = ld_raw<T, VEC>(r + col);
            }
        }
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            const int col = (i * tpr + lane) * VEC;
            if (col < d.D) {
                if (has_res) {
#pragma unroll
                    for (int j = 0; j < VEC; j++) from_f(to_f(a[i].e[j]) + to_f(c[i].e[j]), a[i].e[j]);
                    if (d.tot) *reinterpret_cast<Raw<T, VEC>*>((T*)d.tot + row * d.ld_tot + col) = a[i];
                }
#pragma unroll
                for (int j = 0; j < VEC; j++) v[i][j] = to_f(a[i].e[j]);
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
        if ((i * tpr + lane) * VEC < d.D) {
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                v[i][j] -= mean;
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
        const int col = (i * tpr + lane) * VEC;
        if (col < d.D) {
            float w[VEC], b[VEC];
            Raw<T, VEC> o;
            if (d.w) ld_f<VEC>(d.w + col, w);
            if (d.b) ld_f<VEC>(d.b + col, b);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const float h = v[i][j] * rstd;
                from_f(fmaf(h, d.w ? w[j] : 1.0f, d.b ? b[j] : 0.0f), o.e[j]);
            }
            *reinterpret_cast<Raw<T, VEC>*>(y + col) = o;
        }
    }
}

// Backward.  Blocks walk rows with the grid's stride.  A row stays in registers as it is in memory (bf16: half
// the registers), the normalised entries are computed twice; where registers allow it (PRE) the next row's loads
// are issued before this row's sums.
template <typename T, int VEC, int NCH, bool BLOCK>
struct LnBwd {
    static constexpr int E = NCH * VEC;
    static constexpr bool PRE = !BLOCK && E * (int)sizeof(T) <= 32;
    static constexpr int MIN_BLOCKS = BLOCK ? 1 : E <= 16 ? 2 : 1;
};
template <typename T, int VEC, int NCH, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 32 * LN_WARPS, (LnBwd<T, VEC, NCH, BLOCK>::MIN_BLOCKS))
ln_bwd_kernel(const LnDesc d) {
    constexpr bool PRE = LnBwd<T, VEC, NCH, BLOCK>::PRE;
    extern __shared__ float dynsh[];   // BLOCK: dw, db sums [2][D]; else [2][D] to add the warps in
    __shared__ float sh[32];
    const int lane = BLOCK ? threadIdx.x : (threadIdx.x & 31);
    const int warp = threadIdx.x >> 5;
    const int tpr = BLOCK ? blockDim.x : 32;
    const long long first = BLOCK ? (long long)blockIdx.x : (long long)blockIdx.x * LN_WARPS + warp;
    const long long step = BLOCK ? (long long)gridDim.x : (long long)gridDim.x * LN_WARPS;
    constexpr int NA = BLOCK ? 1 : NCH;
    float aw[NA][VEC], ab[NA][VEC];
    if constexpr (BLOCK) {
        for (int i = threadIdx.x; i < 2 * d.D; i += blockDim.x) dynsh[i] = 0.0f;
        __syncthreads();
    } else {
#pragma unroll
        for (int i = 0; i < NA; i++)
#pragma unroll
            for (int j = 0; j < VEC; j++) aw[i][j] = ab[i][j] = 0.0f;
    }
    struct Row {
        Raw<T, VEC> s[NCH], dy[NCH], t[NCH];
        float mean, rstd;
    };
    auto load = [&](long long row, Row& r) {
        const T* s = (const T*)d.x + row * d.ld_x;
        const T* dy = (const T*)d.dy + row * d.ld_dy;
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            const int col = (i * tpr + lane) * VEC;
            if (col < d.D) {
                r.s[i] = ld_raw<T, VEC>(s + col);
                r.dy[i] = ld_raw<T, VEC>(dy + col);
            }
        }
        if (d.dtot) {
            const T* t = (const T*)d.dtot + row * d.ld_dtot;
#pragma unroll
            for (int i = 0; i < NCH; i++) {
                const int col = (i * tpr + lane) * VEC;
                if (col < d.D) r.t[i] = ld_raw<T, VEC>(t + col);
            }
        }
        r.mean = d.mean[row];
        r.rstd = d.rstd[row];
    };
    Row cur, nxt;
    if (PRE && first < d.rows) load(first, cur);
    for (long long row = first; row < d.rows; row += step) {
        if (!PRE) load(row, cur);
        // dx may be dy or dtotal: the next row belongs to these threads alone, nobody writes it before they read it
        if (PRE && row + step < d.rows) load(row + step, nxt);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            const int col = (i * tpr + lane) * VEC;
            if (col < d.D) {
                float w[VEC];
                if (d.w) ld_f<VEC>(d.w + col, w);
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const float xh = (to_f(cur.s[i].e[j]) - cur.mean) * cur.rstd;
                    const float dy = to_f(cur.dy[i].e[j]);
                    if constexpr (BLOCK) {
                        dynsh[col + j] += dy * xh;
                        dynsh[d.D + col + j] += dy;
                    } else {
                        aw[i][j] = fmaf(dy, xh, aw[i][j]);
                        ab[i][j] += dy;
                    }
                    const float g = d.w ? dy * w[j] : dy;
                    s1 += g;
                    s2 = fmaf(g, xh, s2);
                }
            }
        }
        s1 = row_sum<BLOCK>(s1, sh) / (float)d.D;
        s2 = row_sum<BLOCK>(s2, sh) / (float)d.D;
        T* dx = (T*)d.dx + row * d.ld_dx;
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            const int col = (i * tpr + lane) * VEC;
            if (col < d.D && d.dx) {
                float w[VEC];
                if (d.w) ld_f<VEC>(d.w + col, w);
                Raw<T, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const float xh = (to_f(cur.s[i].e[j]) - cur.mean) * cur.rstd;
                    const float dy = to_f(cur.dy[i].e[j]);
                    float v = cur.rstd * ((d.w ? dy * w[j] : dy) - s1 - xh * s2);
                    if (d.dtot) v += to_f(cur.t[i].e[j]);
                    from_f(v, o.e[j]);
                }
                *reinterpret_cast<Raw<T, VEC>*>(dx + col) = o;
            }
        }
        if (PRE) cur = nxt;
    }
    if (!d.part) return;
    float* part = d.part + (size_t)blockIdx.x * 2 * d.D;
    if constexpr (BLOCK) {
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * d.D; i += blockDim.x) part[i] = dynsh[i];
    } else {
        for (int k = 0; k < LN_WARPS; k++) {   // the warps add in order
            if (warp == k) {
#pragma unroll
                for (int i = 0; i < NA; i++) {
                    const int col = (i * tpr + lane) * VEC;
                    if (col < d.D) {
#pragma unroll
                        for (int j = 0; j < VEC; j++) {
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

// dw[c], db[c] (+)= sum over the blocks' partial sums, in order: 32 columns per
// block, 8 interleaved runs of blocks each, the runs added in order.
__global__ void ln_reduce_kernel(const float* __restrict__ part, int nb, int D, float* __restrict__ dw,
                                 float* __restrict__ db, int accumulate) {
    __shared__ float sh[8][33];
    const int c = blockIdx.x * 32 + threadIdx.x, g = threadIdx.y;
    float v = 0.0f;
    if (c < 2 * D)
        for (int b = g; b < nb; b += 8) v += part[(size_t)b * 2 * D + c];
    sh[g][threadIdx.x] = v;
    __syncthreads();
    if (g == 0 && c < 2 * D) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) s += sh[k][threadIdx.x];
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

// vector form: every row of every tensor starts on 16 bytes
template <typename T>
bool vec_ok(const LnDesc& d, bool bwd) {
    const int V = 16 / (int)sizeof(T);
    if (d.D % V || !aligned16(d.x) || d.ld_x % V || !aligned16(d.w)) return false;
    if (bwd) return aligned16(d.dy) && d.ld_dy % V == 0 && aligned16(d.dtot) && (!d.dtot || d.ld_dtot % V == 0) &&
                    aligned16(d.dx) && (!d.dx || d.ld_dx % V == 0);
    return aligned16(d.b) && aligned16(d.res) && (!d.res || d.ld_res % V == 0) && aligned16(d.tot) &&
           (!d.tot || d.ld_tot % V == 0) && aligned16(d.y) && d.ld_y % V == 0;
}

// Blocks of the backward: enough to fill the device once (two warp blocks per SM, one long-row block), no
// more than there are rows: the partial sums of dw and db grow with them.
int bwd_blocks(long long rows, int D) {
    const long long cap = D <= LN_WARP_D ? 2LL * sm_count() : (long long)sm_count();
    const long long want = D <= LN_WARP_D ? (rows + LN_WARPS - 1) / LN_WARPS : rows;
    return (int)(want < cap ? (want > 0 ? want : 1) : cap);
}
int block_threads(int D) {   // 16 entries per thread
    int t = ((D + 15) / 16 + 31) & ~31;
    return t < 64 ? 64 : t;
}

template <typename T, int VEC, int NCH, bool BLOCK>
cudaError_t fwd_go(const LnDesc& d, cudaStream_t st) {
    const long long blocks = BLOCK ? d.rows : (d.rows + LN_WARPS - 1) / LN_WARPS;
    ln_fwd_kernel<T, VEC, NCH, BLOCK><<<(unsigned)blocks, BLOCK ? block_threads(d.D) : 32 * LN_WARPS, 0, st>>>(d);
    return cudaGetLastError();
}
template <typename T, int VEC, int NCH, bool BLOCK>
cudaError_t bwd_go(const LnDesc& d, cudaStream_t st) {
    const size_t sm = (size_t)2 * d.D * sizeof(float);
    if (sm > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(ln_bwd_kernel<T, VEC, NCH, BLOCK>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm);
        if (e != cudaSuccess) return e;
    }
    ln_bwd_kernel<T, VEC, NCH, BLOCK><<<bwd_blocks(d.rows, d.D), BLOCK ? block_threads(d.D) : 32 * LN_WARPS, sm,
                                        st>>>(d);
    return cudaGetLastError();
}

template <typename T, int VEC, bool BWD>
cudaError_t pick(const LnDesc& d, cudaStream_t st) {
    if (d.D > LN_WARP_D) {
        if constexpr (BWD) return bwd_go<T, VEC, 16 / VEC, true>(d, st);
        else return fwd_go<T, VEC, 16 / VEC, true>(d, st);
    }
    // entries per lane: 8, 16 or 32
#define KMB_LN_GO(E)                                                  \
    {                                                                 \
        if constexpr (BWD) return bwd_go<T, VEC, E / VEC, false>(d, st); \
        else return fwd_go<T, VEC, E / VEC, false>(d, st);            \
    }
    if (d.D <= 256) KMB_LN_GO(8)
    if (d.D <= 512) KMB_LN_GO(16)
    KMB_LN_GO(32)
#undef KMB_LN_GO
}
template <bool BWD>
cudaError_t dispatch(const LnDesc& d, int dtype, cudaStream_t st) {
    if (dtype == KMB_DTYPE_BF16) {
        if (vec_ok<__nv_bfloat16>(d, BWD)) return pick<__nv_bfloat16, 8, BWD>(d, st);
        return pick<__nv_bfloat16, 1, BWD>(d, st);
    }
    if (vec_ok<float>(d, BWD)) return pick<float, 4, BWD>(d, st);
    return pick<float, 1, BWD>(d, st);
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
    return (size_t)bwd_blocks(p->rows, (int)p->D) * 2 * p->D;
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
    LnDesc d{};
    d.rows = p->rows; d.D = (int)p->D; d.eps = p->eps;
    d.x = s; d.ld_x = p->residual ? or_d(p->ld_total, p->D) : or_d(p->ld_x, p->D);
    d.dy = g->dy; d.dtot = g->dtotal; d.dx = g->dx; d.w = p->w; d.mean = p->mean; d.rstd = p->rstd;
    d.ld_dy = or_d(g->ld_dy, p->D); d.ld_dtot = or_d(g->ld_dtotal, p->D); d.ld_dx = or_d(g->ld_dx, p->D);
    d.part = wgrad ? ws : nullptr;
    cudaError_t e = dispatch<true>(d, p->dtype, st);
    if (e == cudaSuccess && wgrad) {
        ln_reduce_kernel<<<(unsigned)((2 * p->D + 31) / 32), dim3(32, 8), 0, st>>>(
            ws, bwd_blocks(p->rows, (int)p->D), (int)p->D, g->dw, g->db, g->accumulate);
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? 0 : set_cuda_error("kmb_layernorm_backward", e);
}

}  // extern "C"
