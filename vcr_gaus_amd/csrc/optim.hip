// Optimizer operators over many tensors at once (no counterpart in the reference, which trains with torch.optim.Adam):
//   AdamW, moments in 32 bits or in 8 bits (blocks of 256 with a power-of-two scale each), fp32 / bf16 / fp16 parameters,
//   optional fp32 masters, step counters on the device;  the 2-norm of many gradients;  codes <-> values of the 8-bit moments.
//
//   t = step, g = grad * grad_scale * coef, coef = min(1, max_norm / (norm + 1e-6)), norm = ||grad * grad_scale|| over all tensors
//   m' = b1 m + (1 - b1) g;  v' = b2 v + (1 - b2) g^2      (each product and sum rounded to fp32: the 8-bit codes are then a
//                                                           function of the inputs alone, whatever the compiler would fuse)
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// 8-bit moments.  For a block of 256 consecutive elements, s = max(1, exponent field of the largest finite |m'|) (8 bits):
//   m code = sign | (bits(|m'| 2^(14 - s)) + r_m) >> 20      4 exponent + 3 mantissa bits; 0x7F = not a number
//   v code =        (bits(v' 2^(30 - s))   + r_v) >> 20      5 + 3 bits, at least 1 where v' > 0 (no division by eps alone);
//                                                            0xFF = not a number
// The scaling is by a power of two, so the float's own exponent field IS the code's (its denormals the code's), and the largest
// binade stays one below the top: rounding up cannot leave the format.  r is random, 16 bits at position 4 plus the half of
// the lowest: stochastic rounding, without which a moment whose relative change per step (1 - b2 = 0.001) is below half a code
// step (2^-4) would never move.  Values keep their codes when a block's scale changes, except at the bottom of the range.
#include "vcr_common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include <new>

namespace {

#define VCR_OPT_BLOCK 256          // elements that share a scale
#define VCR_OPT_TENSORS 352        // tensors and ...
#define VCR_OPT_GROUPS 14          // ... hyper-parameter groups per launch: both travel in the kernel arguments (4 KB)
#define VCR_OPT_NORM_TENSORS 192   // tensors per launch of the norm kernel
#define VCR_OPT_PAIRS 200          // tensors per launch of the code <-> value kernels
#define VCR_OPT_NORM_BLOCKS 2048
#define NORM_CHUNK 16384

struct Group { double lr, wd, log_b1, log_b2; const float* lr_dev; float eps, b1, omb1, b2, omb2; int pad; };
struct StepPack { const void* g[VCR_OPT_TENSORS]; Group group[VCR_OPT_GROUPS]; };
struct PairPack { const void* a[VCR_OPT_PAIRS]; const void* b[VCR_OPT_PAIRS]; };
struct NormPack { const void* g[VCR_OPT_NORM_TENSORS]; long long n[VCR_OPT_NORM_TENSORS]; uint32_t start[VCR_OPT_NORM_TENSORS + 1]; };
static_assert(sizeof(StepPack) <= 4000 && sizeof(NormPack) <= 4000 && sizeof(PairPack) <= 4000, "kernel arguments are 4 KB at most");

struct Coef { float decay, step_size, inv_sqrt_bc2, eps, b1, omb1, b2, omb2; };
struct Clip { float gscale; int skip; };       // of a clipped step, written by the finish kernel

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __hip_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load1(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(__hip_bfloat16* p, float x) { *p = __float2bfloat16(x); }
__device__ __forceinline__ void store1(__half* p, float x) { *p = __float2half(x); }

// V consecutive elements of an aligned array, V = 4 or 8
template <int V> struct Vec { float x[V]; };
template <int V> __device__ __forceinline__ Vec<V> loadv(const float* p) {
    Vec<V> r;
#pragma unroll
    for (int k = 0; k < V; k += 4) {
        const f4 q = *reinterpret_cast<const f4*>(p + k);
        r.x[k] = q.x; r.x[k + 1] = q.y; r.x[k + 2] = q.z; r.x[k + 3] = q.w;
    }
    return r;
}
__device__ __forceinline__ void widen(uint32_t w, float* x, const __hip_bfloat16*) {
    x[0] = __uint_as_float(w << 16); x[1] = __uint_as_float(w & 0xFFFF0000u);
}
__device__ __forceinline__ void widen(uint32_t w, float* x, const __half*) {
    x[0] = __half2float(__ushort_as_half((unsigned short)(w & 0xFFFFu))); x[1] = __half2float(__ushort_as_half((unsigned short)(w >> 16)));
}
__device__ __forceinline__ uint32_t narrow(const float* x, const __hip_bfloat16*) {
    return (uint32_t)__bfloat16_as_ushort(__float2bfloat16(x[0])) | (uint32_t)__bfloat16_as_ushort(__float2bfloat16(x[1])) << 16;
}
__device__ __forceinline__ uint32_t narrow(const float* x, const __half*) {
    return (uint32_t)__half_as_ushort(__float2half(x[0])) | (uint32_t)__half_as_ushort(__float2half(x[1])) << 16;
}
template <int V, typename T> __device__ __forceinline__ Vec<V> loadv(const T* p) {
    Vec<V> r;
    if constexpr (V == 8) {
        const u4 q = *reinterpret_cast<const u4*>(p);
#pragma unroll
        for (int k = 0; k < 4; ++k) widen(q[k], r.x + 2 * k, p);
    } else {
        const u2 q = *reinterpret_cast<const u2*>(p);
#pragma unroll
        for (int k = 0; k < 2; ++k) widen(q[k], r.x + 2 * k, p);
    }
    return r;
}
template <int V> __device__ __forceinline__ void storev(float* p, const Vec<V>& r) {
#pragma unroll
    for (int k = 0; k < V; k += 4) *reinterpret_cast<f4*>(p + k) = f4{r.x[k], r.x[k + 1], r.x[k + 2], r.x[k + 3]};
}
template <int V, typename T> __device__ __forceinline__ void storev(T* p, const Vec<V>& r) {
    if constexpr (V == 8) {
        u4 q;
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = narrow(r.x + 2 * k, p);
        *reinterpret_cast<u4*>(p) = q;
    } else {
        u2 q;
#pragma unroll
        for (int k = 0; k < 2; ++k) q[k] = narrow(r.x + 2 * k, p);
        *reinterpret_cast<u2*>(p) = q;
    }
}
__device__ __forceinline__ bool aligned(const void* p, uint32_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

__device__ __forceinline__ void moments_one(float& m, float& v, float g, const Coef& c) {
#pragma clang fp contract(off)
    m = m * c.b1 + g * c.omb1;
    v = v * c.b2 + (g * g) * c.omb2;
}
// sqrt(v) to 1 ulp also for v below 2^-96, where the instruction alone loses bits
__device__ __forceinline__ float root(float v) {
    const bool small = v < 0x1p-96f;
    const float r = __builtin_amdgcn_sqrtf(small ? v * 0x1p+32f : v);
    return small ? r * 0x1p-16f : r;
}
// square root and reciprocal are the instructions' own 1 ulp: 2e-7 of the update, which itself is rounded into p.  (A denominator
// below 2^-126 -- eps under 1e-38 and no gradient ever -- or above 2^126 takes the division.)
__device__ __forceinline__ float param_one(float p, float m, float v, const Coef& c) {
    const float d = root(v) * c.inv_sqrt_bc2 + c.eps;
    const float q = d >= 0x1p-126f && d <= 0x1p+126f ? m * __builtin_amdgcn_rcpf(d) : m / d;
    return p * c.decay - c.step_size * q;
}

// 32-bit mix (constants found by a search for even avalanche over counters and random words)
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x582C52E9u;
    x = (x ^ (x >> 15)) * 0x1B156CA9u;
    return x ^ (x >> 16);
}
// the random word of an element: `key` = mix32 of (seed, step, tensor, block); one more multiplication spreads the lane
#define LANE_STEP 0x9E3779B1u
__device__ __forceinline__ uint32_t element_word(uint32_t key, uint32_t j_step) {
    uint32_t x = key ^ j_step;
    x = (x ^ (x >> 16)) * 0x582C52E9u;
    return x ^ (x >> 15);
}

#define M_TOP 14
#define V_TOP 30
#define INF_BITS 0x7F800000u
__device__ __forceinline__ float decode_m(uint32_t c, int s) {
    const float x = ldexpf(__uint_as_float((c & 0x7Fu) << 20), s - M_TOP);
    return __uint_as_float(((c & 0x7Fu) == 0x7Fu ? 0x7FC00000u : __float_as_uint(x)) | ((c & 0x80u) << 24));
}
__device__ __forceinline__ float decode_v(uint32_t c, int s) {
    return c == 0xFFu ? __uint_as_float(0x7FC00000u) : ldexpf(__uint_as_float(c << 20), s - V_TOP);
}
__device__ __forceinline__ uint32_t encode_m(float m, int s, uint32_t r) {
    const uint32_t b = __float_as_uint(m), a = b & 0x7FFFFFFFu;
    const uint32_t c = a >= INF_BITS ? 0x7Fu : (__float_as_uint(ldexpf(__uint_as_float(a), M_TOP - s)) + r) >> 20;
    return c | (b >> 24 & 0x80u);
}
__device__ __forceinline__ uint32_t encode_v(float v, int s, uint32_t r) {
    const uint32_t a = __float_as_uint(v) & 0x7FFFFFFFu;
    if (a >= INF_BITS) return 0xFFu;
    const uint32_t c = (__float_as_uint(ldexpf(__uint_as_float(a), V_TOP - s)) + r) >> 20;
    return c == 0u && a != 0u ? 1u : c;
}
__device__ __forceinline__ uint32_t random_m(uint32_t x) { return (x >> 12 & 0xFFFF0u) | 8u; }
__device__ __forceinline__ uint32_t random_v(uint32_t x) { return (x << 4 & 0xFFFF0u) | 8u; }
// largest finite magnitude as float bits (0 for what is not finite)
__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t a = __float_as_uint(x) & 0x7FFFFFFFu;
    return a >= INF_BITS ? 0u : a;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    for (int d = 32; d >= 1; d >>= 1) { const uint32_t y = __shfl_xor(x, d); x = x > y ? x : y; }
    return x;
}
__device__ __forceinline__ int scale_of(uint32_t bits) { const int s = (int)(bits >> 23); return s > 1 ? s : 1; }

// ---- norm -------------------------------------------------------------------------------------------------------
// The sum of squares runs in fp64: neither an fp32 gradient near 1e38 nor 1e9 small ones leave its range, and one partial per
// workgroup, summed in a fixed order, makes the result the same from run to run (no atomics).
__device__ __forceinline__ double block_sum(double x, double* lds) {
    for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

struct Piece { int tensor; long long off; uint32_t cnt; };
__device__ __forceinline__ Piece piece_of(const NormPack& pk, int n, uint32_t chunk, uint32_t c) {
    int lo = 0, hi = n - 1;                    // the tensor whose chunks hold c
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pk.start[mid] <= c) lo = mid; else hi = mid - 1;
    }
    const long long off = (long long)(c - pk.start[lo]) * chunk, left = pk.n[lo] - off;
    return {lo, off, left < (long long)chunk ? (uint32_t)left : chunk};
}
// elements in front of the first 16-byte boundary
template <typename T> __device__ __forceinline__ uint32_t head_of(const T* p, uint32_t cnt) {
    const uint32_t h = (uint32_t)((16u - ((uintptr_t)p & 15u)) & 15u) / sizeof(T);
    return h < cnt ? h : cnt;
}

template <typename T>
__global__ void __launch_bounds__(256) norm_kernel(NormPack pk, int n, uint32_t chunk, double* __restrict__ partials) {
    __shared__ double lds[4];
    constexpr int V = 16 / sizeof(T);
    double sum[V] = {};
    for (uint32_t c = blockIdx.x; c < pk.start[n]; c += gridDim.x) {
        const Piece q = piece_of(pk, n, chunk, c);
        const T* g = (const T*)pk.g[q.tensor] + q.off;
        const uint32_t head = head_of(g, q.cnt), vecs = (q.cnt - head) / V, tail = head + vecs * V;
        if (threadIdx.x < head) { const double x = (double)load1(g + threadIdx.x); sum[0] += x * x; }
        if (threadIdx.x < q.cnt - tail) { const double x = (double)load1(g + tail + threadIdx.x); sum[0] += x * x; }
        const T* body = g + head;
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < vecs; i += 256) {
            const Vec<V> x = loadv<V>(body + (size_t)i * V);
#pragma unroll
            for (int k = 0; k < V; ++k) { const double y = (double)x.x[k]; sum[k] += y * y; }
        }
    }
#pragma unroll
    for (int k = 1; k < V; ++k) sum[0] += sum[k];
    const double total = block_sum(sum[0], lds);
    if (threadIdx.x == 0) partials[blockIdx.x] = total;
}

__device__ __forceinline__ double sum_partials(const double* __restrict__ partials, int n, double* lds) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += partials[i];
    return block_sum(s, lds);
}

// norm = sqrt(sum) |scale|; with `clip`: the factor of a clipped step, and skip where the norm is not finite in fp32
__global__ void __launch_bounds__(256) finish_kernel(const double* __restrict__ partials, int n, double scale, double max_norm,
                                                     float* __restrict__ out, Clip* __restrict__ clip) {
    __shared__ double lds[4];
    const float norm = (float)(sqrt(sum_partials(partials, n, lds)) * fabs(scale));
    if (threadIdx.x != 0) return;
    if (out) *out = norm;
    if (clip) {
        const double q = max_norm / ((double)norm + 1e-6);
        clip->gscale = q < 1.0 ? (float)(scale * q) : (float)scale;
        clip->skip = (__float_as_uint(norm) & 0x7FFFFFFFu) >= INF_BITS;
    }
}

// g *= min(1, max_norm / (norm + 1e-6)); a norm that is not finite leaves NaN or zero as the formula says
template <typename T>
__global__ void __launch_bounds__(256) scale_kernel(NormPack pk, int n, uint32_t chunk, const float* __restrict__ norm, double max_norm) {
    constexpr int V = 16 / sizeof(T);
    const double q = max_norm / ((double)*norm + 1e-6);
    const float f = q > 1.0 ? 1.f : (float)q;
    if (f == 1.f) return;
    for (uint32_t c = blockIdx.x; c < pk.start[n]; c += gridDim.x) {
        const Piece q = piece_of(pk, n, chunk, c);
        T* g = (T*)pk.g[q.tensor] + q.off;
        const uint32_t head = head_of(g, q.cnt), vecs = (q.cnt - head) / V, tail = head + vecs * V;
        if (threadIdx.x < head) store1(g + threadIdx.x, load1(g + threadIdx.x) * f);
        if (threadIdx.x < q.cnt - tail) store1(g + tail + threadIdx.x, load1(g + tail + threadIdx.x) * f);
        T* body = g + head;
        for (uint32_t i = threadIdx.x; i < vecs; i += 256) {
            Vec<V> x = loadv<V>(body + (size_t)i * V);
#pragma unroll
            for (int k = 0; k < V; ++k) x.x[k] *= f;
            storev<V>(body + (size_t)i * V, x);
        }
    }
}

// ---- what every workgroup of an update does first -------------------------------------------------------------------------
// Step counters live on the device (a captured step replays, a skipped one does not count) and one launch does it all, so each
// workgroup forms its tensor's factors itself, in fp64, from the counter: lanes 0 and 1 of a wave share one expm1.  The counter
// may move only when every workgroup of the tensor has read it: each draws a ticket after its read, the last one writes.
struct Work { const void* g; uint32_t cnt; long long off; int step; float gs; };

__device__ __forceinline__ float from_lane(float x, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane)); }

__device__ __forceinline__ Coef coef_of(const Group& G, int t) {
    const int odd = threadIdx.x & 1;
    const double bc = -expm1((double)t * (odd ? G.log_b2 : G.log_b1));           // 1 - b^t
    const double lr = G.lr_dev ? (double)*G.lr_dev : G.lr;
    const float f = odd ? (float)(1.0 / sqrt(bc)) : (float)(lr / bc);
    Coef c;
    c.step_size = from_lane(f, 0);
    c.inv_sqrt_bc2 = from_lane(f, 1);
    c.decay = (float)(1.0 - lr * G.wd);
    c.eps = G.eps; c.b1 = G.b1; c.omb1 = G.omb1; c.b2 = G.b2; c.omb2 = G.omb2;
    return c;
}

// reads the counter, then counts this workgroup in; -> the step this update is
__device__ __forceinline__ int enter(const VcrOptimTensor& R, uint32_t nchunks) {
    __shared__ int step;
    if (threadIdx.x == 0) {
        int* counter = R.step;
        uint32_t* arrived = R.arrived;
        const int t = __hip_atomic_load(counter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        step = t + 1;
        if (nchunks == 1) {
            *counter = t + 1;
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::"v"(t) : "memory");              // (the read is done before the ticket is drawn)
            if (__hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nchunks - 1) {
                __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(counter, t + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
    }
    __syncthreads();
    return step;
}

// ---- update, moments in 32 bits --------------------------------------------------------------------------------------
template <typename T, bool MASTER>
__global__ void __launch_bounds__(256) adamw_kernel(const VcrOptimTensor* __restrict__ tensors, const uint2* __restrict__ chunks,
                                                    uint32_t chunk, const Clip* __restrict__ clip, float gscale, StepPack pk,
                                                    int t0, int g0) {
    constexpr int V = 16 / sizeof(T);
    const uint2 cw = chunks[blockIdx.x];
    const T* g = (const T*)pk.g[cw.x - t0];
    if (!g || (clip && clip->skip)) return;
    const VcrOptimTensor& R = tensors[cw.x];
    const float gs = clip ? clip->gscale : gscale;
    const long long off = (long long)cw.y * chunk, left = R.numel - off;
    const uint32_t cnt = left < (long long)chunk ? (uint32_t)left : chunk;
    const Coef c = coef_of(pk.group[R.group - g0], enter(R, (uint32_t)((R.numel + chunk - 1) / chunk)));
    T* p = (T*)R.p + off;
    float* mst = MASTER ? R.master + off : nullptr;
    float *m = (float*)R.m + off, *v = (float*)R.v + off;
    g += off;
    uint32_t done = 0;
    if (aligned(g, 16) && aligned(p, 16) && aligned(m, 16) && aligned(v, 16) && (!MASTER || aligned(mst, 16))) {
        done = cnt / V * V;
        for (uint32_t i = threadIdx.x * V; i < done; i += 256 * V) {
            const Vec<V> gg = loadv<V>(g + i);
            Vec<V> mm = loadv<V>(m + i), vv = loadv<V>(v + i), x;
            if constexpr (MASTER) x = loadv<V>(mst + i); else x = loadv<V>(p + i);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                moments_one(mm.x[k], vv.x[k], gg.x[k] * gs, c);
                x.x[k] = param_one(x.x[k], mm.x[k], vv.x[k], c);
            }
            storev<V>(m + i, mm);
            storev<V>(v + i, vv);
            if constexpr (MASTER) storev<V>(mst + i, x);
            storev<V>(p + i, x);
        }
    }
    for (uint32_t i = done + threadIdx.x; i < cnt; i += 256) {
        float mm = m[i], vv = v[i];
        moments_one(mm, vv, load1(g + i) * gs, c);
        const float x = param_one(MASTER ? mst[i] : load1(p + i), mm, vv, c);
        m[i] = mm; v[i] = vv;
        if (MASTER) mst[i] = x;
        store1(p + i, x);
    }
}

// ---- update, moments in 8 bits: one wave per block of 256, four consecutive elements per lane ---------------------------
template <typename T>
__device__ __forceinline__ Vec<4> load_some(const T* p, uint32_t i, uint32_t cnt, bool whole) {
    if (whole) return loadv<4>(p + i);
    Vec<4> r;
#pragma unroll
    for (int k = 0; k < 4; ++k) r.x[k] = i + k < cnt ? load1(p + i + k) : 0.f;
    return r;
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, uint32_t i, uint32_t cnt, bool whole, const Vec<4>& r) {
    if (whole) { storev<4>(p + i, r); return; }
#pragma unroll
    for (int k = 0; k < 4; ++k) if (i + k < cnt) store1(p + i + k, r.x[k]);
}
__device__ __forceinline__ uint32_t codes_some(const uint8_t* p, uint32_t i, uint32_t cnt, bool whole) {
    if (whole) return *reinterpret_cast<const uint32_t*>(p + i);
    uint32_t r = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) if (i + k < cnt) r |= (uint32_t)p[i + k] << (8 * k);
    return r;
}
__device__ __forceinline__ void store_codes(uint8_t* p, uint32_t i, uint32_t cnt, bool whole, uint32_t r) {
    if (whole) { *reinterpret_cast<uint32_t*>(p + i) = r; return; }
#pragma unroll
    for (int k = 0; k < 4; ++k) if (i + k < cnt) p[i + k] = (uint8_t)(r >> (8 * k));
}

template <typename T, bool MASTER>
__global__ void __launch_bounds__(256) adamw8_kernel(const VcrOptimTensor* __restrict__ tensors, const uint2* __restrict__ chunks,
                                                     uint32_t chunk, const Clip* __restrict__ clip, float gscale, StepPack pk,
                                                     int t0, int g0, uint32_t seed) {
    const uint2 cw = chunks[blockIdx.x];
    const T* g = (const T*)pk.g[cw.x - t0];
    if (!g || (clip && clip->skip)) return;
    const VcrOptimTensor& R = tensors[cw.x];
    const float gs = clip ? clip->gscale : gscale;
    const long long off = (long long)cw.y * chunk, left = R.numel - off;
    const uint32_t cnt = left < (long long)chunk ? (uint32_t)left : chunk;
    const int step = enter(R, (uint32_t)((R.numel + chunk - 1) / chunk));
    const Coef c = coef_of(pk.group[R.group - g0], step);
    T* p = (T*)R.p + off;
    float* mst = MASTER ? R.master + off : nullptr;
    uint8_t *mc = (uint8_t*)R.m + off, *vc = (uint8_t*)R.v + off;
    g += off;
    const bool al = aligned(g, 4 * sizeof(T)) && aligned(p, 4 * sizeof(T)) && aligned(mc, 4) && aligned(vc, 4) && (!MASTER || aligned(mst, 16));
    const uint32_t j0 = (threadIdx.x & 63) * 4;
    const uint32_t key = mix32(mix32(mix32(seed) + (uint32_t)step) + (uint32_t)R.index);
    const uint32_t blk0 = (uint32_t)(off / VCR_OPT_BLOCK);
    const uint8_t *ms = R.m_scale + blk0, *vs = R.v_scale + blk0;
    for (uint32_t b = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); b * VCR_OPT_BLOCK < cnt; b += 4) {
        const uint32_t i = b * VCR_OPT_BLOCK + j0;
        const bool whole = al && (b + 1) * VCR_OPT_BLOCK <= cnt;
        const int sm = ms[b], sv = vs[b];
        const Vec<4> gg = load_some(g, i, cnt, whole);
        Vec<4> x;
        if constexpr (MASTER) x = load_some(mst, i, cnt, whole); else x = load_some(p, i, cnt, whole);
        uint32_t cm = codes_some(mc, i, cnt, whole), cv = codes_some(vc, i, cnt, whole);
        float mm[4], vv[4];
        uint32_t mb = 0, vb = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            mm[k] = decode_m(cm >> (8 * k) & 255u, sm);
            vv[k] = decode_v(cv >> (8 * k) & 255u, sv);
            moments_one(mm[k], vv[k], gg.x[k] * gs, c);
            x.x[k] = param_one(x.x[k], mm[k], vv[k], c);
            mb = max(mb, finite_bits(mm[k]));
            vb = max(vb, finite_bits(vv[k]));
        }
        if constexpr (MASTER) store_some(mst, i, cnt, whole, x);
        store_some(p, i, cnt, whole, x);
        const int nm = scale_of(wave_max(mb)), nv = scale_of(wave_max(vb));
        const uint32_t bkey = mix32(key + blk0 + b);
        cm = cv = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t w = element_word(bkey, (j0 + k) * LANE_STEP);
            cm |= encode_m(mm[k], nm, random_m(w)) << (8 * k);
            cv |= encode_v(vv[k], nv, random_v(w)) << (8 * k);
        }
        store_codes(mc, i, cnt, whole, cm);
        store_codes(vc, i, cnt, whole, cv);
        if (j0 == 0) { R.m_scale[blk0 + b] = (uint8_t)nm; R.v_scale[blk0 + b] = (uint8_t)nv; }
    }
}

// ---- codes -> values, values -> codes (to the nearest, ties to even) ------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) decode_kernel(const VcrOptimTensor* __restrict__ tensors, const uint2* __restrict__ chunks,
                                                     uint32_t chunk, PairPack out, int t0) {
    const uint2 cw = chunks[blockIdx.x];
    const VcrOptimTensor& R = tensors[cw.x];
    const long long off = (long long)cw.y * chunk;
    const long long left = R.numel - off;
    const uint32_t cnt = left < (long long)chunk ? (uint32_t)left : chunk;
    T *mo = (T*)out.a[cw.x - t0], *vo = (T*)out.b[cw.x - t0];
    for (uint32_t i = threadIdx.x; i < cnt; i += 256) {
        const long long e = off + i;
        if (mo) store1(mo + e, decode_m(((const uint8_t*)R.m)[e], R.m_scale[e / VCR_OPT_BLOCK]));
        if (vo) store1(vo + e, decode_v(((const uint8_t*)R.v)[e], R.v_scale[e / VCR_OPT_BLOCK]));
    }
}

__device__ __forceinline__ uint32_t nearest_m(float m, int s) {
    const uint32_t y = __float_as_uint(ldexpf(fabsf(m), M_TOP - s));
    return encode_m(m, s, 0x7FFFFu + (y >> 20 & 1u));
}
__device__ __forceinline__ uint32_t nearest_v(float v, int s) {
    const uint32_t y = __float_as_uint(ldexpf(fabsf(v), V_TOP - s));
    return encode_v(v, s, 0x7FFFFu + (y >> 20 & 1u));
}
__global__ void __launch_bounds__(256) encode_kernel(const VcrOptimTensor* __restrict__ tensors, const uint2* __restrict__ chunks,
                                                     uint32_t chunk, PairPack in, int t0) {
    const uint2 cw = chunks[blockIdx.x];
    const VcrOptimTensor& R = tensors[cw.x];
    const long long off = (long long)cw.y * chunk;
    const long long left = R.numel - off;
    const uint32_t cnt = left < (long long)chunk ? (uint32_t)left : chunk;
    const float *mi = (const float*)in.a[cw.x - t0] + off, *vi = (const float*)in.b[cw.x - t0] + off;
    uint8_t *mc = (uint8_t*)R.m + off, *vc = (uint8_t*)R.v + off;
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t b = threadIdx.x >> 6; b * VCR_OPT_BLOCK < cnt; b += 4) {
        const long long blk = off / VCR_OPT_BLOCK + b;
        uint32_t mb = 0, vb = 0;
        for (uint32_t i = b * VCR_OPT_BLOCK + lane; i < cnt && i < (b + 1) * VCR_OPT_BLOCK; i += 64) {
            mb = max(mb, finite_bits(mi[i]));
            vb = max(vb, finite_bits(vi[i]));
        }
        const int nm = scale_of(wave_max(mb)), nv = scale_of(wave_max(vb));
        for (uint32_t i = b * VCR_OPT_BLOCK + lane; i < cnt && i < (b + 1) * VCR_OPT_BLOCK; i += 64) {
            mc[i] = (uint8_t)nearest_m(mi[i], nm);
            vc[i] = (uint8_t)nearest_v(vi[i], nv);
        }
        if (lane == 0) { R.m_scale[blk] = (uint8_t)nm; R.v_scale[blk] = (uint8_t)nv; }
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------
inline int64_t chunks_of(int64_t numel, int64_t chunk) { return (numel + chunk - 1) / chunk; }
inline size_t plan_head(int n) { return vcr_align(sizeof(VcrOptimTensor) * (size_t)n); }
inline bool chunk_ok(int chunk) { return chunk >= 1024 && chunk % 1024 == 0 && chunk <= (1 << 20); }
inline const uint2* plan_chunks(const void* plan, int n) { return (const uint2*)((const char*)plan + plan_head(n)); }

// checks that the calls on a plan share; returns the number of chunks, -1 with an error set
int64_t plan_check(const char* who, const void* plan, int n, const int64_t* numel, int chunk) {
    if (!plan || !numel || n < 1 || !chunk_ok(chunk)) { vcr_set_error("%s: plan, numel or chunk is missing or out of range", who); return -1; }
    int64_t total = 0;
    for (int k = 0; k < n; ++k) {
        if (numel[k] < 0) { vcr_set_error("%s: tensor %d has numel %lld", who, k, (long long)numel[k]); return -1; }
        total += chunks_of(numel[k], chunk);
    }
    if (total > 0x7FFFFFFF) { vcr_set_error("%s: %lld chunks", who, (long long)total); return -1; }
    return total;
}

// runs `launch` over the non-empty tensors of one type, in packs that fit the kernel arguments
template <typename F>
int each_norm_pack(int n, const void* const* tensors, const int64_t* numel, const int32_t* types, int type, F launch) {
    int k = 0;
    while (k < n) {
        NormPack pk;
        int used = 0;
        int64_t start = 0;
        pk.start[0] = 0;
        for (; k < n && used < VCR_OPT_NORM_TENSORS; ++k) {
            if (numel[k] == 0 || types[k] != type) continue;
            const int64_t c = chunks_of(numel[k], NORM_CHUNK);
            if (start + c > 0x7FFFFFFF) break;
            pk.g[used] = tensors[k];
            pk.n[used] = numel[k];
            start += c;
            pk.start[++used] = (uint32_t)start;
        }
        if (used == 0) {
            if (k < n) { vcr_set_error("tensor %d with %lld elements is too large", k, (long long)numel[k]); return 1; }
            break;
        }
        if (launch(pk, used, (uint32_t)start)) return 1;
    }
    return 0;
}

int list_check(const char* who, int n, const void* const* tensors, const int64_t* numel, const int32_t* types) {
    if (n < 0 || (n > 0 && (!tensors || !numel || !types))) { vcr_set_error("%s: the list of tensors is missing", who); return 1; }
    for (int k = 0; k < n; ++k)
        if (numel[k] < 0 || (numel[k] > 0 && !tensors[k]) || types[k] < 0 || types[k] > VCR_F16) {
            vcr_set_error("%s: tensor %d has numel %lld, pointer %p, type %d", who, k, (long long)numel[k], tensors[k], types[k]);
            return 1;
        }
    return 0;
}

}  // namespace

extern "C" size_t vcr_optim_plan_bytes(int ntensors, const int64_t* numel, int chunk) {
    if (ntensors < 1 || !numel || !chunk_ok(chunk)) return 0;
    size_t total = 0;
    for (int k = 0; k < ntensors; ++k) total += numel[k] > 0 ? (size_t)chunks_of(numel[k], chunk) : 0;
    return plan_head(ntensors) + sizeof(uint2) * total;
}

extern "C" int vcr_optim_plan(int ntensors, const VcrOptimTensor* tensors, int chunk, void* host_plan, size_t bytes) {
    if (ntensors < 1 || !tensors || !host_plan || !chunk_ok(chunk)) { vcr_set_error("vcr_optim_plan: tensors, plan or chunk is missing or out of range"); return 1; }
    size_t total = 0;
    for (int k = 0; k < ntensors; ++k) {
        const VcrOptimTensor& t = tensors[k];
        if (t.numel < 0 || !t.step || !t.arrived || (t.numel > 0 && (!t.p || !t.m || !t.v)) || (!t.m_scale != !t.v_scale)) {
            vcr_set_error("vcr_optim_plan: tensor %d has numel %lld and a pointer missing", k, (long long)t.numel);
            return 1;
        }
        total += (size_t)chunks_of(t.numel, chunk);
    }
    if (total > 0x7FFFFFFF || bytes < plan_head(ntensors) + sizeof(uint2) * total) { vcr_set_error("vcr_optim_plan: %zu bytes for %zu chunks", bytes, total); return 1; }
    VcrOptimTensor* out = (VcrOptimTensor*)host_plan;
    uint2* c = (uint2*)((char*)host_plan + plan_head(ntensors));
    for (int k = 0; k < ntensors; ++k) {
        out[k] = tensors[k];
        const uint32_t nc = (uint32_t)chunks_of(tensors[k].numel, chunk);
        for (uint32_t i = 0; i < nc; ++i) *c++ = make_uint2((uint32_t)k, i);
    }
    return 0;
}

extern "C" int vcr_adamw_step(const VcrAdamWStep* args, void* stream) {
    if (!args) { vcr_set_error("vcr_adamw_step: args is NULL"); return 1; }
    const VcrAdamWStep& a = *args;
    if (a.ntensors == 0) return 0;
    if (plan_check("vcr_adamw_step", a.plan, a.ntensors, a.numel, a.chunk) < 0) return 1;
    if (!a.grads || !a.groups || !a.group_of || a.ngroups < 1 || a.param_type < 0 || a.param_type > VCR_F16 ||
        (a.state_bits != 32 && a.state_bits != 8) || (a.masters && a.param_type == VCR_F32)) {
        vcr_set_error("vcr_adamw_step: inconsistent arguments");
        return 1;
    }
    for (int k = 0; k < a.ngroups; ++k) {
        const VcrOptimGroup& g = a.groups[k];
        if (!(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0 && g.eps >= 0.0)) {
            vcr_set_error("vcr_adamw_step: group %d has beta1 %g, beta2 %g, eps %g", k, g.beta1, g.beta2, g.eps);
            return 1;
        }
    }
    for (int k = 0; k < a.ntensors; ++k)
        if (a.group_of[k] < 0 || a.group_of[k] >= a.ngroups || (k && a.group_of[k] < a.group_of[k - 1])) {
            vcr_set_error("vcr_adamw_step: tensor %d is in group %d of %d (groups must ascend)", k, a.group_of[k], a.ngroups);
            return 1;
        }
    hipStream_t st = (hipStream_t)stream;
    const VcrOptimTensor* tensors = (const VcrOptimTensor*)a.plan;
    const uint2* chunks = plan_chunks(a.plan, a.ntensors);
    const Clip* clip = (const Clip*)a.clip;
    for (int t0 = 0, t1 = 0; t0 < a.ntensors; t0 = t1) {
        StepPack pk = {};
        int64_t nchunks = 0;
        bool any = false;
        const int g0 = a.group_of[t0];
        for (; t1 < a.ntensors && t1 - t0 < VCR_OPT_TENSORS && a.group_of[t1] - g0 < VCR_OPT_GROUPS; ++t1) {
            pk.g[t1 - t0] = a.grads[t1];
            nchunks += chunks_of(a.numel[t1], a.chunk);
            any |= a.grads[t1] != nullptr && a.numel[t1] > 0;
        }
        for (int k = g0; k <= a.group_of[t1 - 1]; ++k) {
            const VcrOptimGroup& g = a.groups[k];
            pk.group[k - g0] = {g.lr, g.weight_decay, log(g.beta1), log(g.beta2), g.lr_dev, (float)g.eps,
                                (float)g.beta1, (float)(1.0 - g.beta1), (float)g.beta2, (float)(1.0 - g.beta2), 0};
        }
        if (any) {
            const dim3 grid((uint32_t)nchunks), block(256);
            const float gs = (float)a.grad_scale;
#define LAUNCH32(T, M) hipLaunchKernelGGL((adamw_kernel<T, M>), grid, block, 0, st, tensors, chunks, (uint32_t)a.chunk, clip, gs, pk, t0, g0)
#define LAUNCH8(T, M) hipLaunchKernelGGL((adamw8_kernel<T, M>), grid, block, 0, st, tensors, chunks, (uint32_t)a.chunk, clip, gs, pk, t0, g0, a.seed)
#define LAUNCH(T, M) do { if (a.state_bits == 32) LAUNCH32(T, M); else LAUNCH8(T, M); } while (0)
            if (a.param_type == VCR_F32) LAUNCH(float, false);
            else if (a.param_type == VCR_BF16) { if (a.masters) LAUNCH(__hip_bfloat16, true); else LAUNCH(__hip_bfloat16, false); }
            else { if (a.masters) LAUNCH(__half, true); else LAUNCH(__half, false); }
#undef LAUNCH
#undef LAUNCH8
#undef LAUNCH32
        }
        chunks += nchunks;
    }
    VCR_HIP_CHECK(hipGetLastError());
    return 0;
}

static int pairs_call(const char* who, int n, const void* plan, const int64_t* numel, int chunk, const void* const* a, const void* const* b,
                      int type, bool encode, hipStream_t st) {
    if (n == 0) return 0;
    if (plan_check(who, plan, n, numel, chunk) < 0) return 1;
    if (!a || !b || type < 0 || type > VCR_F16) { vcr_set_error("%s: inconsistent arguments", who); return 1; }
    const VcrOptimTensor* tensors = (const VcrOptimTensor*)plan;
    const uint2* chunks = plan_chunks(plan, n);
    for (int t0 = 0; t0 < n; t0 += VCR_OPT_PAIRS) {
        PairPack pk = {};
        int64_t nchunks = 0;
        for (int k = 0; k < VCR_OPT_PAIRS && t0 + k < n; ++k) {
            pk.a[k] = a[t0 + k];
            pk.b[k] = b[t0 + k];
            if (encode && numel[t0 + k] > 0 && (!pk.a[k] || !pk.b[k])) { vcr_set_error("%s: values of tensor %d are missing", who, t0 + k); return 1; }
            nchunks += chunks_of(numel[t0 + k], chunk);
        }
        if (nchunks > 0) {
            const dim3 grid((uint32_t)nchunks), block(256);
            if (encode) hipLaunchKernelGGL(encode_kernel, grid, block, 0, st, tensors, chunks, (uint32_t)chunk, pk, t0);
            else if (type == VCR_F32) hipLaunchKernelGGL(decode_kernel<float>, grid, block, 0, st, tensors, chunks, (uint32_t)chunk, pk, t0);
            else if (type == VCR_BF16) hipLaunchKernelGGL(decode_kernel<__hip_bfloat16>, grid, block, 0, st, tensors, chunks, (uint32_t)chunk, pk, t0);
            else hipLaunchKernelGGL(decode_kernel<__half>, grid, block, 0, st, tensors, chunks, (uint32_t)chunk, pk, t0);
        }
        chunks += nchunks;
    }
    VCR_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int vcr_moments8_decode(int ntensors, const void* plan, const int64_t* numel, int chunk, void* const* exp_avg,
                                   void* const* exp_avg_sq, int type, void* stream) {
    return pairs_call("vcr_moments8_decode", ntensors, plan, numel, chunk, exp_avg, exp_avg_sq, type, false, (hipStream_t)stream);
}
extern "C" int vcr_moments8_encode(int ntensors, const void* plan, const int64_t* numel, int chunk, const float* const* exp_avg,
                                   const float* const* exp_avg_sq, void* stream) {
    return pairs_call("vcr_moments8_encode", ntensors, plan, numel, chunk, (const void* const*)exp_avg, (const void* const*)exp_avg_sq, VCR_F32,
                      true, (hipStream_t)stream);
}

extern "C" int vcr_grad_norm_partials(int ntensors, const int64_t* numel) {
    if (ntensors < 1 || !numel) return 1;
    int64_t chunks = 0;
    for (int k = 0; k < ntensors; ++k) chunks += numel[k] > 0 ? chunks_of(numel[k], NORM_CHUNK) : 0;
    const int64_t packs = ntensors / VCR_OPT_NORM_TENSORS + 3 + chunks / 0x40000000;     // (a pack ends with its type)
    const int64_t most = packs * VCR_OPT_NORM_BLOCKS;
    return (int)(chunks < most ? chunks + 1 : most);
}

extern "C" int vcr_grad_norm(int ntensors, const void* const* tensors, const int64_t* numel, const int32_t* types, double* partials,
                             int capacity, double grad_scale, double max_norm, float* norm, void* clip, void* stream) {
    if (list_check("vcr_grad_norm", ntensors, tensors, numel, types)) return 1;
    if (!partials || (!norm && !clip)) { vcr_set_error("vcr_grad_norm: partials or norm is NULL"); return 1; }
    if (clip && !(max_norm > 0.0)) { vcr_set_error("vcr_grad_norm: max_norm is %g", max_norm); return 1; }
    hipStream_t st = (hipStream_t)stream;
    int used_partials = 0;
    for (int type = VCR_F32; type <= VCR_F16; ++type) {
        const int rc = each_norm_pack(ntensors, tensors, numel, types, type, [&](const NormPack& pk, int used, uint32_t chunks) {
            const int blocks = chunks < VCR_OPT_NORM_BLOCKS ? (int)chunks : VCR_OPT_NORM_BLOCKS;
            if (used_partials + blocks > capacity) { vcr_set_error("vcr_grad_norm: room for %d partial sums is too little", capacity); return 1; }
            const dim3 grid(blocks), block(256);
            double* out = partials + used_partials;
            if (type == VCR_F32) hipLaunchKernelGGL(norm_kernel<float>, grid, block, 0, st, pk, used, NORM_CHUNK, out);
            else if (type == VCR_BF16) hipLaunchKernelGGL(norm_kernel<__hip_bfloat16>, grid, block, 0, st, pk, used, NORM_CHUNK, out);
            else hipLaunchKernelGGL(norm_kernel<__half>, grid, block, 0, st, pk, used, NORM_CHUNK, out);
            used_partials += blocks;
            return 0;
        });
        if (rc) return 1;
    }
    hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(256), 0, st, partials, used_partials, grad_scale, max_norm, norm, (Clip*)clip);
    VCR_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int vcr_clip_gradients(int ntensors, void* const* tensors, const int64_t* numel, const int32_t* types, const float* norm,
                                  double max_norm, void* stream) {
    if (list_check("vcr_clip_gradients", ntensors, tensors, numel, types)) return 1;
    if (!norm || !(max_norm > 0.0)) { vcr_set_error("vcr_clip_gradients: norm is NULL or max_norm is %g", max_norm); return 1; }
    hipStream_t st = (hipStream_t)stream;
    for (int type = VCR_F32; type <= VCR_F16; ++type) {
        const int rc = each_norm_pack(ntensors, tensors, numel, types, type, [&](const NormPack& pk, int used, uint32_t chunks) {
            const dim3 grid(chunks < 4096 ? chunks : 4096), block(256);
            if (type == VCR_F32) hipLaunchKernelGGL(scale_kernel<float>, grid, block, 0, st, pk, used, NORM_CHUNK, norm, max_norm);
            else if (type == VCR_BF16) hipLaunchKernelGGL(scale_kernel<__hip_bfloat16>, grid, block, 0, st, pk, used, NORM_CHUNK, norm, max_norm);
            else hipLaunchKernelGGL(scale_kernel<__half>, grid, block, 0, st, pk, used, NORM_CHUNK, norm, max_norm);
            return 0;
        });
        if (rc) return 1;
    }
    VCR_HIP_CHECK(hipGetLastError());
    return 0;
}
