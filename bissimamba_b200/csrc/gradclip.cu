// gradclip.cu -- global gradient norm over many tensors, and clipping by it
// (include/kmamba_clip.h).
//
// Two passes over the data, each one launch per GC_LIST tensors: the sum of
// squares, then the scaling.  Both are bound by HBM, so all they do is keep wide
// loads in flight: a tensor is cut into chunks of 16-byte pieces (plus the few
// entries before its first 16-byte boundary and behind its last), the grid walks
// the chunks of all tensors, and the tensors' table travels as a kernel
// argument, so a call copies nothing and allocates nothing.
//
// The sum: squares of the entries of 16-byte pieces are added in fp32 and each
// partial sum of 32 goes into a 64-bit one; where that partial sum is outside
// the range in which fp32 squares are exact to rounding (an overflow, or entries
// whose squares are subnormal) it is taken again in 64 bits.  One partial sum per
// block, added in block order by every block of the second pass: no atomics.
//
// A block takes a run of chunks, the second pass from the last to the first:
// what the first pass read last is still in L2 when the second begins.  It does nothing for a
// tensor that is scaled in place by 1.
//
// Measured: 170 M gradients, half of them bf16 (510 MB), clipped into other
// buffers in 275 us: 5.6 TB/s over three passes of the data (sum 103 us, the
// rest scaling); a 12-layer model's 3.5 M (14 MB, in L2) in 10 us of device time, two
// launches' latency.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cmath>
#include <cstdint>
#include "../../include/kmamba_clip.h"
#include "kmb_launch.cuh"

namespace kmb {
int set_error(const char* msg);
int set_cuda_error(const char* where, cudaError_t e);
void clear_error();

namespace {

constexpr int GC_LIST = 256;          // tensors per launch
constexpr int GC_THREADS = 256;
constexpr int GC_VPT = 8;             // 16-byte pieces per thread and chunk
constexpr long long GC_CHUNK = (long long)GC_THREADS * GC_VPT;   // pieces per chunk
constexpr int GC_MAX_BLOCKS = 2048;

struct GcTensor {
    const void* in;
    void* out;
    long long n;
};
template <int CAP>
struct GcList {
    GcTensor t[CAP];
    int first[CAP + 1];   // first chunk of each tensor
    unsigned char bf16[CAP];
    int count;
};

__device__ __forceinline__ int head_of(const void* p, int esz, long long n) {
    const int h = (int)(((16 - ((uintptr_t)p & 15)) & 15) / esz);
    return (long long)h < n ? h : (int)n;
}
// chunks of this block: a run, so that the tensor of the next chunk is this one's or the one after
__device__ __forceinline__ int run_start(int chunks, int b) { return (int)((long long)chunks * b / gridDim.x); }
template <int CAP>
__device__ __forceinline__ int find_tensor(const GcList<CAP>& l, int chunk) {
    int a = 0, b = l.count;   // last tensor whose first chunk is <= chunk and that has chunks
    while (b - a > 1) {
        const int m = (a + b) >> 1;
        if (l.first[m] <= chunk) a = m;
        else b = m;
    }
    return a;
}
__device__ __forceinline__ void unpack(const uint4& r, bool bf, float (&v)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    if (bf) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = __uint_as_float(w[i]);
            v[4 + i] = 0.0f;
        }
    }
}
__device__ __forceinline__ float load1(const void* p, long long i, bool bf) {
    return bf ? __bfloat162float(((const __nv_bfloat16*)p)[i]) : ((const float*)p)[i];
}

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < GC_THREADS / 32; i++) s += sh[i];
    return s;
}

// squares of `cnt` 16-byte pieces: fp32 within the call, 64 bits across calls
__device__ __forceinline__ double squares(const uint4* r, int cnt, bool bf) {
    float s = 0.0f;
    uint32_t any = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (k >= cnt) break;
        float v[8];
        unpack(r[k], bf, v);
        any |= r[k].x | r[k].y | r[k].z | r[k].w;
#pragma unroll
        for (int i = 0; i < 4; i++) s = fmaf(v[i], v[i], s);
        if (bf) {
#pragma unroll
            for (int i = 4; i < 8; i++) s = fmaf(v[i], v[i], s);
        }
    }
    // between 2^-60 and 2^120 no square that matters was rounded to a subnormal and none overflowed (an
    // entry whose square is below 2^-126 is then below 2^-33 of the sum's root)
    if (!any || (s > 8.7e-19f && s < 1.3e36f)) return (double)s;
    double q = 0.0;
    for (int k = 0; k < cnt; k++) {
        float v[8];
        unpack(r[k], bf, v);
        for (int i = 0; i < 8; i++) q = fma((double)v[i], (double)v[i], q);
    }
    return q;
}

template <int CAP>
__global__ void __launch_bounds__(GC_THREADS)
gc_norm_kernel(const __grid_constant__ GcList<CAP> l, double* __restrict__ part) {
    __shared__ double sh[GC_THREADS / 32];
    double acc = 0.0;
    pdl_release();
    const int chunks = l.first[l.count];
    const int c0 = run_start(chunks, blockIdx.x), c1 = run_start(chunks, blockIdx.x + 1);
    int t = find_tensor(l, c0);
    for (int c = c0; c < c1; c++) {
        while (l.first[t + 1] <= c) t++;
        const GcTensor& x = l.t[t];
        const bool bf = l.bf16[t] != 0;
        const int esz = bf ? 2 : 4, vec = 16 / esz;
        const int head = head_of(x.in, esz, x.n);
        const long long pieces = (x.n - head) / vec;
        const uint4* body = (const uint4*)((const char*)x.in + (size_t)head * esz);
        const long long p0 = (long long)(c - l.first[t]) * GC_CHUNK;
        uint4 r[GC_VPT];
        if (p0 + GC_CHUNK <= pieces) {
#pragma unroll
            for (int k = 0; k < GC_VPT; k++) r[k] = __ldg(body + p0 + k * GC_THREADS + threadIdx.x);
        } else {
#pragma unroll
            for (int k = 0; k < GC_VPT; k++) {
                const long long p = p0 + k * GC_THREADS + threadIdx.x;
                r[k] = p < pieces ? __ldg(body + p) : make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int k = 0; k < GC_VPT; k += 4) acc += squares(r + k, 4, bf);
        if (c == l.first[t]) {   // the tensor's ends
            const long long tail = head + pieces * vec;
            if (threadIdx.x < head) {
                const double v = load1(x.in, threadIdx.x, bf);
                acc = fma(v, v, acc);
            }
            if (tail + threadIdx.x < x.n) {
                const double v = load1(x.in, tail + threadIdx.x, bf);
                acc = fma(v, v, acc);
            }
        }
    }
    const double s = block_sum(acc, sh);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <int CAP>
__global__ void __launch_bounds__(GC_THREADS)
gc_scale_kernel(const __grid_constant__ GcList<CAP> l, const double* part, int nparts, float max_norm, float* result) {
    __shared__ double sh[GC_THREADS / 32];
    pdl_wait();
    double s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += GC_THREADS) s += part[i];
    const double norm = sqrt(block_sum(s, sh));
    float coef = 1.0f;
    if (norm > (double)max_norm && norm <= 1.7976931348623157e308) coef = (float)((double)max_norm / norm);
    if (result && blockIdx.x == 0 && threadIdx.x == 0) {
        result[0] = (float)norm;
        result[1] = coef;
    }
    const int chunks = l.first[l.count];
    const int c0 = run_start(chunks, blockIdx.x), c1 = run_start(chunks, blockIdx.x + 1);
    int t = c1 > c0 ? find_tensor(l, c1 - 1) : 0;
    for (int c = c1 - 1; c >= c0; c--) {
        while (l.first[t] > c) t--;
        const GcTensor& x = l.t[t];
        if (!x.out || (coef == 1.0f && x.out == x.in)) continue;
        const bool bf = l.bf16[t] != 0;
        const int esz = bf ? 2 : 4, vec = 16 / esz;
        const int head = head_of(x.in, esz, x.n);
        const long long pieces = (x.n - head) / vec;
        const char* body = (const char*)x.in + (size_t)head * esz;
        char* obody = (char*)x.out + (size_t)head * esz;
        const bool wide = ((uintptr_t)obody & 15) == 0;
        const long long p0 = (long long)(c - l.first[t]) * GC_CHUNK;
        uint4 r[GC_VPT];
#pragma unroll
        for (int k = 0; k < GC_VPT; k++) {
            const long long p = p0 + k * GC_THREADS + threadIdx.x;
            r[k] = p < pieces ? *((const uint4*)body + p) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < GC_VPT; k++) {
            const long long p = p0 + k * GC_THREADS + threadIdx.x;
            if (p >= pieces) continue;
            float v[8];
            unpack(r[k], bf, v);
            if (coef != 1.0f) {   // by 1 an entry is copied as it is, infinities and NaN among them
                uint32_t w[4];
                if (bf) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i] * coef, v[2 * i + 1] * coef);
                        w[i] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] = __float_as_uint(v[i] * coef);
                }
                r[k] = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (wide) {
                *((uint4*)obody + p) = r[k];
            } else {
                const uint32_t w[4] = {r[k].x, r[k].y, r[k].z, r[k].w};
                if (bf) {
                    uint16_t* o = (uint16_t*)obody + p * 8;
#pragma unroll
                    for (int i = 0; i < 8; i++) o[i] = (uint16_t)(w[i >> 1] >> ((i & 1) * 16));
                } else {
                    uint32_t* o = (uint32_t*)obody + p * 4;
#pragma unroll
                    for (int i = 0; i < 4; i++) o[i] = w[i];
                }
            }
        }
        if (c == l.first[t]) {
            const long long tail = head + pieces * vec;
            auto one = [&](long long i) {
                const float v = load1(x.in, i, bf) * coef;
                if (bf) ((__nv_bfloat16*)x.out)[i] = __float2bfloat16_rn(v);
                else ((float*)x.out)[i] = v;
            };
            if (threadIdx.x < head) one(threadIdx.x);
            if (tail + threadIdx.x < x.n) one(tail + threadIdx.x);
        }
    }
}

int sm_count() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n;
}
int grid_of(int chunks) {
    const int most = 6 * sm_count() < GC_MAX_BLOCKS ? 6 * sm_count() : GC_MAX_BLOCKS;
    return chunks < most ? (chunks > 0 ? chunks : 1) : most;
}

// One launch's table from list entries [i0, ...): returns how many entries it took, 0 if a tensor is too long.
template <int CAP>
long fill(GcList<CAP>& l, const KMBGradTensor* ts, long i0, long n) {
    long i = i0;
    int k = 0;
    long long chunk = 0;
    for (; i < n && k < CAP; i++) {
        if (ts[i].n == 0) continue;
        const int vec = ts[i].dtype == KMB_DTYPE_BF16 ? 8 : 4;
        const long long c = (ts[i].n / vec + GC_CHUNK) / GC_CHUNK;   // at least one: the ends belong to the first
        if (chunk + c > 0x7fffffffLL) break;
        l.t[k] = {ts[i].in, ts[i].out, ts[i].n};
        l.bf16[k] = ts[i].dtype == KMB_DTYPE_BF16;
        l.first[k] = (int)chunk;
        chunk += c;
        k++;
    }
    l.count = k;
    l.first[k] = (int)chunk;
    return i - i0;
}

template <int CAP>
cudaError_t clip_all(const KMBGradTensor* ts, long n, float max_norm, float* result, double* part, long max_parts,
                     cudaStream_t st, bool* too_long) {
    GcList<CAP> l;
    int nparts = 0, single = 0;
    cudaError_t e = cudaSuccess;
    for (long i = 0; i < n;) {
        const long took = fill(l, ts, i, n);
        if (took == 0) { *too_long = true; return cudaSuccess; }
        if (l.count) {
            const int g = grid_of(l.first[l.count]);
            if (nparts + g > max_parts) return cudaErrorInvalidValue;
            gc_norm_kernel<CAP><<<g, GC_THREADS, 0, st>>>(l, part + nparts);
            single++;
            nparts += g;
        }
        i += took;
    }
    bool first = true;
    for (long i = 0; i < n || first;) {   // an empty list still reports its norm
        const long took = fill(l, ts, i, n);
        // only the launch right behind the one sum may be set up while that runs
        if ((l.count || first) && e == cudaSuccess)
            e = launch(gc_scale_kernel<CAP>, dim3((unsigned)grid_of(l.first[l.count])), dim3(GC_THREADS), 0, st,
                       first && single == 1, l, (const double*)part, nparts, max_norm, first ? result : (float*)nullptr);
        first = false;
        i += took;
    }
    return e == cudaSuccess ? cudaGetLastError() : e;
}

constexpr int GC_SMALL = 64;
long launches_of(long n) { return n <= GC_SMALL ? 1 : (n + GC_LIST - 1) / GC_LIST; }

}  // namespace
}  // namespace kmb

using namespace kmb;

extern "C" {

size_t kmb_grad_clip_workspace_floats(long n_tensors) {
    // one 64-bit partial sum per block and launch; a launch ends early where its tensors exceed 2^31 chunks,
    // which needs more memory than the device has
    return n_tensors < 0 ? 0 : (size_t)launches_of(n_tensors > 0 ? n_tensors : 1) * GC_MAX_BLOCKS * 2;
}

int kmb_grad_clip(const KMBGradTensor* ts, long n, float max_norm, float* result, float* ws, void* stream) {
    clear_error();
    if (n < 0 || (n > 0 && !ts)) return set_error("kmb_grad_clip: invalid list");
    if (!(max_norm > 0.0f)) return set_error("kmb_grad_clip: max_norm must be above 0");
    if (!ws || ((uintptr_t)ws & 7)) return set_error("kmb_grad_clip: an 8-byte aligned workspace is required");
    for (long i = 0; i < n; i++) {
        if (ts[i].dtype != KMB_DTYPE_F32 && ts[i].dtype != KMB_DTYPE_BF16) return set_error("kmb_grad_clip: unknown dtype");
        if (ts[i].n < 0 || (ts[i].n > 0 && !ts[i].in)) return set_error("kmb_grad_clip: invalid tensor");
        const uintptr_t m = ts[i].dtype == KMB_DTYPE_BF16 ? 1 : 3;
        if (((uintptr_t)ts[i].in & m) || ((uintptr_t)ts[i].out & m))
            return set_error("kmb_grad_clip: a tensor is not aligned to its elements");
    }
    if ((uintptr_t)result & 3) return set_error("kmb_grad_clip: result is not aligned to its elements");
    bool too_long = false;
    const long parts = launches_of(n > 0 ? n : 1) * GC_MAX_BLOCKS;
    cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e = n <= GC_SMALL
                        ? clip_all<GC_SMALL>(ts, n, max_norm, result, (double*)ws, parts, st, &too_long)
                        : clip_all<GC_LIST>(ts, n, max_norm, result, (double*)ws, parts, st, &too_long);
    if (too_long) return set_error("kmb_grad_clip: a tensor is too long");
    return e == cudaSuccess ? 0 : set_cuda_error("kmb_grad_clip", e);
}

}  // extern "C"
