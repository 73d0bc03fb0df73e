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
#include <string.h>

namespace {

#define VCR_OPT_BLOCK 256          // elements that share a scale
#define VCR_OPT_CHUNK 4096         // elements per entry of a plan
// Threads per workgroup; four elements each and no loop in the 32-bit update: a workgroup reads, computes, writes and is gone, so that
// the ones in flight work on neighbouring memory (1 M Gaussians: 289 us with four rounds of 1024 elements per workgroup, 279 us
// with one; 1024 threads 291 us).
#define VCR_OPT_THREADS 256
#define VCR_OPT_TENSORS 352        // tensors and ...
#define VCR_OPT_GROUPS 14          // ... hyper-parameter groups per launch: both travel in the kernel arguments (4 KB)
#define VCR_OPT_LAUNCH_CHUNKS 4194303   // plan entries per launch: a launch has fewer than 2^32 threads, 1024 an entry at most
#define VCR_OPT_NORM_TENSORS 192   // tensors per launch of the norm kernel
#define VCR_OPT_PAIRS 200          // tensors per launch of the code <-> value kernels
// The norm's workgroups stride over chunks (800 M fp32 elements: 459 us with 1024 workgroups, 469 with 2048, 468 with 4096).
#define VCR_OPT_NORM_BLOCKS 1024
#define NORM_CHUNK 16384
#define NORM_LAUNCH_CHUNKS 0x7FFFFFFF      // of one tensor, and of one launch
// Up to this many chunks in all, of one type: one workgroup and one launch (64 K fp32 elements, 4 chunks: 8.9 instead of 11.8 us from
// Python, 4.8 us either way in a captured graph; 8 chunks 8.9 instead of 12.0, but 8.5 instead of 4.9 captured).
#define VCR_OPT_NORM_ONE 4

struct Group { double lr, wd, log_b1, log_b2; const float* lr_dev; float eps, b1, omb1, b2, omb2; int pad; };
struct StepPack { const void* g[VCR_OPT_TENSORS]; Group group[VCR_OPT_GROUPS]; };
struct PairPack { const void* a[VCR_OPT_PAIRS]; const void* b[VCR_OPT_PAIRS]; };
struct NormPack { const void* g[VCR_OPT_NORM_TENSORS]; long long n[VCR_OPT_NORM_TENSORS]; uint32_t start[VCR_OPT_NORM_TENSORS + 1]; };
static_assert(sizeof(StepPack) <= 4000 && sizeof(NormPack) <= 4000 && sizeof(PairPack) <= 4000, "kernel arguments are 4 KB at most");

struct Coef { float decay, step_size, inv_sqrt_bc2, eps, b1, omb1, b2, omb2; int plain; };
struct Clip { float gscale; int skip; };       // of a clipped step, written by the finish kernel

// Pointers read from memory are generic to the compiler (flat_* accesses, which wait on two counters); these are global.
#define GLOBAL __attribute__((address_space(1)))
template <typename T> __device__ __forceinline__ GLOBAL T* global(T* p) { return (GLOBAL T*)(uintptr_t)p; }

__device__ __forceinline__ float load1(const GLOBAL float* p) { return *p; }
__device__ __forceinline__ float load1(const GLOBAL __hip_bfloat16* p) {
    return __uint_as_float((uint32_t)*(const GLOBAL unsigned short*)p << 16);
}
__device__ __forceinline__ float load1(const GLOBAL __half* p) { return __half2float(__ushort_as_half(*(const GLOBAL unsigned short*)p)); }
__device__ __forceinline__ void store1(GLOBAL float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(GLOBAL __hip_bfloat16* p, float x) {
    *(GLOBAL unsigned short*)p = __bfloat16_as_ushort(__float2bfloat16(x));
}
__device__ __forceinline__ void store1(GLOBAL __half* p, float x) { *(GLOBAL unsigned short*)p = __half_as_ushort(__float2half(x)); }

// Four consecutive elements at any address that the element's type allows: the types below are aligned to one element, and the
// hardware takes such addresses in its 8- and 16-byte accesses as they are.  NT: past the caches' retention, for what a step
// touches once: parameters, gradients, moments (400 M elements 2 079 -> 1 868 us, 302 M bf16 elements with masters 1 599 -> 1 400 us).
typedef float f4a __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4a __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u2a __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u2b __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u1a __attribute__((aligned(1)));
template <bool NT, typename Q> __device__ __forceinline__ Q ldq(const GLOBAL void* p) {
    if constexpr (NT) return __builtin_nontemporal_load((const GLOBAL Q*)p);
    else return *(const GLOBAL Q*)p;
}
template <bool NT, typename Q> __device__ __forceinline__ void stq(GLOBAL void* p, Q q) {
    if constexpr (NT) __builtin_nontemporal_store(q, (GLOBAL Q*)p);
    else *(GLOBAL Q*)p = q;
}
template <int V> struct Vec { float x[V]; };
__device__ __forceinline__ void widen(uint32_t w, float* x, const GLOBAL __hip_bfloat16*) {
    x[0] = __uint_as_float(w << 16); x[1] = __uint_as_float(w & 0xFFFF0000u);
}
__device__ __forceinline__ void widen(uint32_t w, float* x, const GLOBAL __half*) {
    x[0] = __half2float(__ushort_as_half((unsigned short)(w & 0xFFFFu))); x[1] = __half2float(__ushort_as_half((unsigned short)(w >> 16)));
}
__device__ __forceinline__ uint32_t narrow(const float* x, const GLOBAL __hip_bfloat16*) {
    return (uint32_t)__bfloat16_as_ushort(__float2bfloat16(x[0])) | (uint32_t)__bfloat16_as_ushort(__float2bfloat16(x[1])) << 16;
}
__device__ __forceinline__ uint32_t narrow(const float* x, const GLOBAL __half*) {
    return (uint32_t)__half_as_ushort(__float2half(x[0])) | (uint32_t)__half_as_ushort(__float2half(x[1])) << 16;
}
// (V = 4, or as many elements as 16 bytes hold)
template <int V, bool NT, typename T> __device__ __forceinline__ Vec<V> loadv(const GLOBAL T* p) {
    Vec<V> r;
    if constexpr (sizeof(T) == 4) {
        const f4a q = ldq<NT, f4a>(p);
#pragma unroll
        for (int k = 0; k < 4; ++k) r.x[k] = q[k];
    } else if constexpr (V == 8) {
        const u4a q = ldq<NT, u4a>(p);
#pragma unroll
        for (int k = 0; k < 4; ++k) widen(q[k], r.x + 2 * k, p);
    } else {
        const u2a q = ldq<NT, u2a>(p);
#pragma unroll
        for (int k = 0; k < 2; ++k) widen(q[k], r.x + 2 * k, p);
    }
    return r;
}
template <int V, bool NT, typename T> __device__ __forceinline__ void storev(GLOBAL T* p, const Vec<V>& r) {
    if constexpr (sizeof(T) == 4) {
        stq<NT>(p, f4a{r.x[0], r.x[1], r.x[2], r.x[3]});
    } else if constexpr (V == 8) {
        u4a q;
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = narrow(r.x + 2 * k, p);
        stq<NT>(p, q);
    } else {
        u2a q;
#pragma unroll
        for (int k = 0; k < 2; ++k) q[k] = narrow(r.x + 2 * k, p);
        stq<NT>(p, q);
    }
}

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
// Square root and reciprocal are the instructions' own, 1 ulp: 2e-7 of the update, which is itself rounded into p.  (The host refuses
// an eps that is denormal in fp32, so the denominator is 0, normal or infinite.)
__device__ __forceinline__ float param_one(float p, float m, float v, const Coef& c) {
    return p * c.decay - c.step_size * (m * __builtin_amdgcn_rcpf(root(v) * c.inv_sqrt_bc2 + c.eps));
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
__device__ __forceinline__ int scale_of(uint32_t bits) { const int s = (int)(bits >> 23); return s > 1 ? s : 1; }

// ---- norm -------------------------------------------------------------------------------------------------------
// The sum of squares runs in fp64: neither an fp32 gradient near 1e38 nor 1e9 small ones leave its range, and one partial per
// workgroup, summed in a fixed order, makes the result the same from run to run (no atomics).
template <int THREADS> __device__ __forceinline__ double block_sum(double x) {
    __shared__ double lds[THREADS / 64];
    for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
    for (int k = 1; k < THREADS / 64; ++k) x += lds[k];
    return x;
}

// norm = sqrt(sum) |scale|; with `clip`: the factor of a clipped step, and skip where the norm is not finite in fp32
struct Finish { double scale, max_norm; float* out; Clip* clip; };
__device__ __forceinline__ void finish(double sum, const Finish& f) {
    const float norm = (float)(sqrt(sum) * fabs(f.scale));
    if (f.out) *f.out = norm;
    if (f.clip) {
        const double q = f.max_norm / ((double)norm + 1e-6);
        f.clip->gscale = q < 1.0 ? (float)(f.scale * q) : (float)f.scale;
        f.clip->skip = (__float_as_uint(norm) & 0x7FFFFFFFu) >= INF_BITS;
    }
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
// NT: gradients that nothing reads soon again pass the caches (800 M fp32 elements 520 -> 459 us, 7.0 TB/s; 302 M bf16 106 -> 95 us);
// those of a clipped step stay in them for the update behind (75 M fp32 elements, norm and update together: 379 against 420 us).
// ONE: few elements in all, one large workgroup that writes the norm itself: one launch instead of two.
template <typename T, bool NT, bool ONE> constexpr int norm_threads() { return ONE ? 1024 : 256; }
template <typename T, bool NT, bool ONE>
__global__ void __launch_bounds__((norm_threads<T, NT, ONE>())) norm_kernel(NormPack pk, int n, uint32_t chunk, double* __restrict__ partials,
                                                                          Finish f) {
    constexpr int V = 16 / sizeof(T), THREADS = norm_threads<T, NT, ONE>();
    double sum[V] = {};
    for (uint32_t c = blockIdx.x; c < pk.start[n]; c += gridDim.x) {
        const Piece q = piece_of(pk, n, chunk, c);
        const GLOBAL T* g = global((const T*)pk.g[q.tensor]) + q.off;
        const uint32_t vecs = q.cnt / V, tail = vecs * V;
        if (threadIdx.x < q.cnt - tail) { const double x = (double)load1(g + tail + threadIdx.x); sum[0] += x * x; }
#pragma unroll 4
        for (uint32_t i = threadIdx.x; i < vecs; i += THREADS) {
            const Vec<V> x = loadv<V, NT>(g + (size_t)i * V);
#pragma unroll
            for (int k = 0; k < V; ++k) { const double y = (double)x.x[k]; sum[k] += y * y; }
        }
    }
#pragma unroll
    for (int k = 1; k < V; ++k) sum[0] += sum[k];
    const double total = block_sum<THREADS>(sum[0]);
    if (threadIdx.x != 0) return;
    if constexpr (ONE) finish(total, f);
    else partials[blockIdx.x] = total;
}

// (1024 threads, one partial each, take as long: 4.9 us behind a large norm, 1.9 against 1.6 us behind a small one)
__global__ void __launch_bounds__(256) finish_kernel(const double* __restrict__ partials, int n, Finish f) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += partials[i];
    s = block_sum<256>(s);
    if (threadIdx.x == 0) finish(s, f);
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
        GLOBAL T* g = global((T*)pk.g[q.tensor]) + q.off;
        const uint32_t vecs = q.cnt / V, tail = vecs * V;
        if (threadIdx.x < q.cnt - tail) store1(g + tail + threadIdx.x, load1(g + tail + threadIdx.x) * f);
        for (uint32_t i = threadIdx.x; i < vecs; i += 256) {
            Vec<V> x = loadv<V, false>(g + (size_t)i * V);
#pragma unroll
            for (int k = 0; k < V; ++k) x.x[k] *= f;
            storev<V, false>(g + (size_t)i * V, x);
        }
    }
}

// ---- what every workgroup of an update does first -------------------------------------------------------------------------
// Step counters live on the device (a captured step replays, a skipped one does not count) and one launch does it all, so each
// workgroup forms its tensor's factors itself from the counter: its first wave does, lanes 0 and 1 sharing one expm1,
// while the data loads of all waves are in flight.  The counter may move only when every workgroup of the tensor has read
// it: each draws a ticket after its read, the last one writes.
struct Place { uint32_t tensor, part; long long first; };
// Which elements a workgroup takes, 4 ROUNDS per thread; VCR_OPT_CHUNK / (1024 ROUNDS) workgroups share an entry of the plan.
template <int ROUNDS> constexpr uint32_t parts() { return VCR_OPT_CHUNK / (4 * VCR_OPT_THREADS * ROUNDS); }
template <int ROUNDS> __device__ __forceinline__ Place place(const uint2* __restrict__ chunks) {
    const uint2 c = chunks[blockIdx.x / parts<ROUNDS>()];
    const uint32_t part = blockIdx.x % parts<ROUNDS>();
    return {c.x, c.y * parts<ROUNDS>() + part, (long long)c.y * VCR_OPT_CHUNK + part * (4 * VCR_OPT_THREADS * ROUNDS)};
}
__device__ __forceinline__ float from_lane(float x, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane)); }

__device__ __forceinline__ Coef coef_of(const Group& G, int t) {
    // 1 - b^t from the rounded exponent: 1e-7 of the update, like its root and reciprocal
    const int odd = threadIdx.x & 1;
    const float bc = -expm1f((float)((double)t * (odd ? G.log_b2 : G.log_b1)));
    const double lr = G.lr_dev ? (double)*G.lr_dev : G.lr;
    const float f = odd ? 1.f / sqrtf(bc) : (float)lr / bc;
    Coef c;
    c.step_size = from_lane(f, 0);
    c.inv_sqrt_bc2 = from_lane(f, 1);
    c.decay = (float)(1.0 - lr * G.wd);
    c.eps = G.eps; c.b1 = G.b1; c.omb1 = G.omb1; c.b2 = G.b2; c.omb2 = G.omb2;
    // Whether the 8-bit fast path, which divides by the step size, applies: not with a step size of zero, nor where its denominator
    // could leave the normal numbers, whose reciprocal is infinite (m' = 0 would become NaN).  eps / step size is 0 or normal by the
    // test (which has room for the reciprocal's rounding); with eps = 0 the root of a v' of 2^-126 or more (`Fast::guard`), times a
    // factor of 1 or more, over a step size below 2^60 is above 2^-123.  (Formed here once, not in every wave, where it delays the
    // loads: 295 M fp32 elements and their values 1 036 instead of 1 156 us.)
    c.plain = c.step_size > 1e-20f && c.step_size < 0x1p+60f && (c.eps == 0.f || c.eps >= 0x1.01p-126f * c.step_size);
    return c;
}

// Counts this workgroup out (its read of the counter is long done: the factors came from it), at the end, where nothing waits for the
// ticket: drawn before the results are written it costs 3 to 6 %.  Tickets on one address come at 12.5 ns each (a tensor of
// 400 M elements in 195 000 workgroups would take 2.4 ms for them alone, measured), so a tensor with many chunks has 64 first-level
// words, and only the last arrival of each goes to the second level.
#define TICKET_GROUPS 64
#define TICKET_FLAT 64             // up to this many chunks: one level
#define TICKET_STRIDE 16           // words between two tickets: a cache line of their own
__device__ __forceinline__ bool last_of(GLOBAL uint32_t* word, uint32_t of) {
    if (__hip_atomic_fetch_add(word, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != of - 1) return false;
    __hip_atomic_store(word, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}
template <int ROUNDS> __device__ __forceinline__ void leave(const VcrOptimTensor& R, uint32_t* words, const Place& at, int step) {
    if (threadIdx.x != 0) return;
    const uint32_t nchunks = R.numel ? (uint32_t)((R.numel + VCR_OPT_CHUNK - 1) / VCR_OPT_CHUNK) : 1u, n = nchunks * parts<ROUNDS>();
    bool last = true;
    if (n > 1) {
        GLOBAL uint32_t* w = global(words) + (size_t)R.words * TICKET_STRIDE;
        if (nchunks <= TICKET_FLAT) {
            last = last_of(w, n);
        } else {
            const uint32_t g = at.part % TICKET_GROUPS;
            last = last_of(w + (1 + g) * TICKET_STRIDE, (n - g + TICKET_GROUPS - 1) / TICKET_GROUPS) && last_of(w, TICKET_GROUPS);
        }
    }
    if (last) *global(R.step) = step;
}
// the step that this update is, and its factors, the same in every lane; `leave` follows when the results are out
struct Entry { int step; Coef coef; };
__device__ __forceinline__ Entry enter(const VcrOptimTensor& R, const Group& G) {
    __shared__ Entry entry;
    if (threadIdx.x < 64) {
        const int t = *global(R.step) + 1;
        const Coef coef = coef_of(G, t);
        if (threadIdx.x == 0) { entry.step = t; entry.coef = coef; }
    }
    __syncthreads();
    return entry;
}

// ---- update, moments in 32 bits: four consecutive elements per lane ----------------------------------------------------
template <typename T, bool MASTER>
__global__ void __launch_bounds__(VCR_OPT_THREADS) adamw_kernel(const VcrOptimTensor* __restrict__ tensors, const uint2* __restrict__ chunks,
                                                                uint32_t* __restrict__ words, const Clip* __restrict__ clip, float gscale,
                                                                StepPack pk, int t0, int g0) {
    const Place at = place<1>(chunks);
    const GLOBAL T* g = global((const T*)pk.g[at.tensor - t0]);
    if (!g || (clip && clip->skip)) return;
    const VcrOptimTensor& R = tensors[at.tensor];
    const uint32_t group = (uint32_t)(R.group - g0);
    if (group >= VCR_OPT_GROUPS || R.m_scale || (MASTER && !R.master && R.numel)) return;             // (a plan that was made for another call)
    const float gs = clip ? clip->gscale : gscale;
    const long long off = at.first + threadIdx.x * 4, left = R.numel - off;
    GLOBAL T* p = global((T*)R.p) + off;
    GLOBAL float* mst = MASTER ? global(R.master) + off : nullptr;
    GLOBAL float *m = global((float*)R.m) + off, *v = global((float*)R.v) + off;
    g += off;
    Vec<4> gg = {}, mm = {}, vv = {}, x = {};
    if (left >= 4) {
        gg = loadv<4, true>(g);
        mm = loadv<4, true>(m);
        vv = loadv<4, true>(v);
        if constexpr (MASTER) x = loadv<4, true>(mst);
        else x = loadv<4, true>(p);
    } else {
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (k < left) {
                gg.x[k] = load1(g + k); mm.x[k] = m[k]; vv.x[k] = v[k];
                x.x[k] = MASTER ? mst[k] : load1(p + k);
            }
    }
    const Entry e = enter(R, pk.group[group]);
    const Coef c = e.coef;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        moments_one(mm.x[k], vv.x[k], gg.x[k] * gs, c);
        x.x[k] = param_one(x.x[k], mm.x[k], vv.x[k], c);
    }
    if (left >= 4) {
        storev<4, true>(m, mm);
        storev<4, true>(v, vv);
        if constexpr (MASTER) storev<4, true>(mst, x);
        storev<4, true>(p, x);
    } else {
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (k < left) {
                m[k] = mm.x[k]; v[k] = vv.x[k];
                if (MASTER) mst[k] = x.x[k];
                store1(p + k, x.x[k]);
            }
    }
    leave<1>(R, words, at, e.step);
}

// ---- update, moments in 8 bits: one wave per block of 256, four consecutive elements per lane ---------------------------
// Maximum over a wave: within rows of 16 by lane permutations, across the four rows on the scalar side.
template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 15, 15, true); }
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
    x = max(x, dpp<0xB1>(x));          // lanes 1 0 3 2
    x = max(x, dpp<0x4E>(x));          // lanes 2 3 0 1
    x = max(x, dpp<0x141>(x));         // halves of 8 mirrored
    return max(x, dpp<0x140>(x));      // rows of 16 mirrored
}
// (the compiler would take these three to the vector side)
__device__ __forceinline__ uint32_t smax(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("s_max_u32 %0, %1, %2" : "=s"(r) : "s"(a), "s"(b) : "scc");
    return r;
}
__device__ __forceinline__ uint32_t rows_max(uint32_t x) {
    const uint32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16);
    const uint32_t c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
    return smax(smax(a, b), smax(c, d));
}

struct Lane8 { Vec<4> g, x; uint32_t cm, cv; };      // what a lane loads: gradient, parameter, codes
typedef float f2 __attribute__((ext_vector_type(2)));

// byte 3 of four words, in order
__device__ __forceinline__ uint32_t top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0703u), __builtin_amdgcn_perm(b, a, 0x0C0C0703u), 0x05040100u);
}
__device__ __forceinline__ float power(int field) { return __uint_as_float((uint32_t)field << 23); }      // 2^(field - 127), 1 <= field <= 254
// byte K of x at bits 20 ... 27
template <int K> __device__ __forceinline__ float code_bits(uint32_t x, uint32_t twenty) {
    uint32_t r;
    if constexpr (K == 0) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_0" : "=v"(r) : "v"(twenty), "v"(x));
    if constexpr (K == 1) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_1" : "=v"(r) : "v"(twenty), "v"(x));
    if constexpr (K == 2) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_2" : "=v"(r) : "v"(twenty), "v"(x));
    if constexpr (K == 3) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_3" : "=v"(r) : "v"(twenty), "v"(x));
    return __uint_as_float(r);
}
// block exponents for which every power of two below is a normal number, and no value that the codes stand for is denormal
#define M_LOW 40
#define M_HIGH 139
#define V_LOW 40
#define V_HIGH 155

// The factors once more, as the fast path takes them: p' = p decay - m' / (sqrt(v') root + eps), both divided by the step size.
// `guard`: whether eps is so small that a root flushed to zero (v' below 2^-126: the root below 1e-19, 3e-18 with the largest factor
// that b2 = 0.999 gives) could be seen.
struct Fast { float root, eps; bool guard; };
__device__ __forceinline__ Fast fast_of(const Coef& c) {
    const float r = __builtin_amdgcn_rcpf(c.step_size);
    const int eps = __builtin_amdgcn_readfirstlane(__float_as_int(c.eps)), isq = __builtin_amdgcn_readfirstlane(__float_as_int(c.inv_sqrt_bc2));
    return {c.inv_sqrt_bc2 * r, c.eps * r, !(__int_as_float(eps) >= 1e-10f && __int_as_float(isq) < 40.f)};
}

// A whole block of finite numbers of ordinary size: the definition above with its scalings as multiplications by powers of two
// (exact, so that b2 and the scale of v are one factor), the first moment's codes decoded by the hardware (they are OCP e4m3:
// bias 7, code exponent 14 = 2^7), and everything shifted up by 4 so that a code is the top byte of its word.  Returns false, with
// nothing changed, where it does not apply: a code or a moment that is not finite, block exponents out of the ranges above, or,
// where eps is small enough for it to be seen (`guard`), a second moment below 2^-126, which the square root instruction would
// flush.  Its 154 vector instructions, of 196 a block in all, are what bounds the update of 16-bit parameters without masters: in
// 95 % of the cycles one is at work (with masters in 54 %).
__device__ __forceinline__ bool block_fast(Lane8& r, int& sm, int& sv, uint32_t bkey, const uint32_t (&j_step)[4], float gs, const Coef& c,
                                           const Fast& f) {
#pragma clang fp contract(off)
    if (!__builtin_amdgcn_readfirstlane(c.plain) || sm < M_LOW || sm > M_HIGH || sv < V_LOW || sv > V_HIGH) return false;
    // a byte 0x7F / 0xFF among the first moment's codes, a byte 0xFF among the second's
    uint32_t odd = ((r.cm & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
    odd |= ((r.cv & 0x7F7F7F7Fu) + 0x01010101u) & r.cv & 0x80808080u;
    const float m_scale = power(sm - 7), v_scale = power(sv - V_TOP + 127) * c.b2;
    const f2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(r.cm, m_scale, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(r.cm, m_scale, true);
    float m[4] = {lo.x, lo.y, hi.x, hi.y};
    float v[4] = {code_bits<0>(r.cv, 20), code_bits<1>(r.cv, 20), code_bits<2>(r.cv, 20), code_bits<3>(r.cv, 20)};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float g = r.g.x[k] * gs;
        m[k] = m[k] * c.b1 + g * c.omb1;
        v[k] = v[k] * v_scale + (g * g) * c.omb2;
    }
    const float ma = fmaxf(fmaxf(fabsf(m[0]), fabsf(m[1])), fmaxf(fabsf(m[2]), fabsf(m[3])));
    const uint32_t va = max(max(__float_as_uint(v[0]), __float_as_uint(v[1])), max(__float_as_uint(v[2]), __float_as_uint(v[3])));
    const uint32_t mr = row_max(__float_as_uint(ma)), vr = row_max(va);
    const uint32_t mb = rows_max(mr), vb = rows_max(vr);                     // (m' is finite where v' is)
    const int nm = (int)(mb >> 23), nv = (int)(vb >> 23);
    if (nm < M_LOW || nm > M_HIGH || nv < V_LOW || nv > V_HIGH || __any(odd != 0)) return false;
    if (f.guard) {
        bool tiny = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) tiny |= __builtin_amdgcn_classf(v[k], 0x90);               // denormal
        if (__any(tiny)) return false;
    }
    sm = nm;
    sv = nv;
    const float m_up = power(M_TOP - nm + 127), v_up = power(V_TOP - nv + 127);
    uint32_t zm[4], zv[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        {
#pragma clang fp contract(fast)
            const float d = __builtin_amdgcn_sqrtf(v[k]) * f.root + f.eps;
            r.x.x[k] = r.x.x[k] * c.decay - m[k] * __builtin_amdgcn_rcpf(d);
        }
        // 16 r_m and 16 r_v: the word's upper and lower half at bits 8 ... 23, 0x80 below
        const uint32_t w = element_word(bkey, j_step[k]);
        zm[k] = (__float_as_uint(fabsf(m[k]) * m_up) << 4) + __builtin_amdgcn_perm(w, 0x80u, 0x0C070600u);
        // at least code 1 (2^-129) where v' > 0: the middle one of the scaled value, of 2^20 v' -- larger than either, as v_up is
        // 2^-10 at most and the smallest v' is 2^-149; 0 where v' is 0 -- and of code 1
        const float y = __builtin_amdgcn_fmed3f(v[k] * v_up, v[k] * 0x1p+20f, __uint_as_float(1u << 20));
        zv[k] = (__float_as_uint(y) << 4) + __builtin_amdgcn_perm(w, 0x80u, 0x0C050400u);
    }
    const uint32_t sign = top_bytes(__float_as_uint(m[0]), __float_as_uint(m[1]), __float_as_uint(m[2]), __float_as_uint(m[3])) & 0x80808080u;
    r.cm = sign | top_bytes(zm[0], zm[1], zm[2], zm[3]);
    r.cv = top_bytes(zv[0], zv[1], zv[2], zv[3]);
    return true;
}

// Any block: `n` of the lane's four elements exist.
__device__ __forceinline__ void block_any(Lane8& r, int& sm, int& sv, uint32_t bkey, const uint32_t (&j_step)[4], int n, float gs, const Coef& c) {
    float m[4], v[4];
    uint32_t mb = 0, vb = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        m[k] = decode_m(r.cm >> (8 * k) & 255u, sm);
        v[k] = decode_v(r.cv >> (8 * k) & 255u, sv);
        moments_one(m[k], v[k], r.g.x[k] * gs, c);
        r.x.x[k] = param_one(r.x.x[k], m[k], v[k], c);
        if (k < n) { mb = max(mb, finite_bits(m[k])); vb = max(vb, finite_bits(v[k])); }
    }
    sm = scale_of(rows_max(row_max(mb)));
    sv = scale_of(rows_max(row_max(vb)));
    r.cm = r.cv = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t w = element_word(bkey, j_step[k]);
        r.cm |= encode_m(m[k], sm, random_m(w)) << (8 * k);
        r.cv |= encode_v(v[k], sv, random_v(w)) << (8 * k);
    }
}

// One block: addresses of its first elements (the same in every lane: the lane's offset j0 is added by the accesses themselves), how
// many of the lane's four elements exist.
template <typename T> struct Block8 {
    const GLOBAL T* g;
    GLOBAL T* p;
    GLOBAL float* mst;
    GLOBAL uint8_t *mc, *vc;
    bool whole;
    int n;
};
template <typename T, bool MASTER>
__device__ __forceinline__ Lane8 load_block(const Block8<T>& b, uint32_t j0) {
    // (measured both ways in turn on one card, which the kept forms are not alike on: with the non-temporal kind 302 M bf16 elements take
    //  523 instead of 564 us, but fp32 ones, 295 M, 776 instead of 752, and bf16 ones with masters 821 instead of 803; on others the
    //  kept forms take up to 597 and 821 us)
    constexpr bool NT = sizeof(T) == 2 && !MASTER;
    Lane8 r = {};
    if (b.whole) {
        r.g = loadv<4, NT>(b.g + j0);
        if constexpr (MASTER) r.x = loadv<4, true>(b.mst + j0);
        else r.x = loadv<4, NT>((const GLOBAL T*)b.p + j0);
        r.cm = ldq<true, u1a>(b.mc + j0);
        r.cv = ldq<true, u1a>(b.vc + j0);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < b.n) {
                r.g.x[k] = load1(b.g + j0 + k);
                r.x.x[k] = MASTER ? b.mst[j0 + k] : load1((const GLOBAL T*)b.p + j0 + k);
                r.cm |= (uint32_t)b.mc[j0 + k] << (8 * k);
                r.cv |= (uint32_t)b.vc[j0 + k] << (8 * k);
            }
    }
    return r;
}
template <typename T, bool MASTER>
__device__ __forceinline__ void store_block(const Block8<T>& b, uint32_t j0, const Lane8& r) {
    if (b.whole) {
        if constexpr (MASTER) storev<4, true>(b.mst + j0, r.x);
        storev<4, true>(b.p + j0, r.x);
        stq<true>(b.mc + j0, (u1a)r.cm);
        stq<true>(b.vc + j0, (u1a)r.cv);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < b.n) {
                if (MASTER) b.mst[j0 + k] = r.x.x[k];
                store1(b.p + j0 + k, r.x.x[k]);
                b.mc[j0 + k] = (uint8_t)(r.cm >> (8 * k));
                b.vc[j0 + k] = (uint8_t)(r.cv >> (8 * k));
            }
    }
}

// Blocks of a wave, one after another.  What every wave does once (addresses, factors) is a third of its instructions with one block:
// 16-bit parameters without masters (10 bytes an element) are bound by instructions and take four (302 M elements 731, 601, 524 us
// with 1, 2, 4 blocks), with masters two (19 M elements in odd sizes 57.5, 49.4, 51.0 us); fp32 (16 bytes) is bound by memory, which
// favours short runs of a workgroup, and takes one (295 M elements 772, 777, 840 us).  Each of these sets on one card, in turn.
template <typename T, bool MASTER> constexpr int blocks8() { return sizeof(T) == 4 ? 1 : MASTER ? 2 : 4; }
template <typename T, bool MASTER>
__global__ void __launch_bounds__(VCR_OPT_THREADS) adamw8_kernel(const VcrOptimTensor* __restrict__ tensors, const uint2* __restrict__ chunks,
                                                                 uint32_t* __restrict__ words, const Clip* __restrict__ clip, float gscale,
                                                                 StepPack pk, int t0, int g0, uint32_t seed) {
    constexpr int BLOCKS = blocks8<T, MASTER>();
    const Place at = place<BLOCKS>(chunks);
    const T* grad = (const T*)pk.g[at.tensor - t0];
    if (!grad || (clip && clip->skip)) return;
    const VcrOptimTensor& R = tensors[at.tensor];
    const uint32_t group = (uint32_t)(R.group - g0);
    if (group >= VCR_OPT_GROUPS || ((!R.m_scale || (MASTER && !R.master)) && R.numel)) return;       // (a plan that was made for another call)
    const float gs = clip ? clip->gscale : gscale;
    const Entry e = enter(R, pk.group[group]);
    const Fast fast = fast_of(e.coef);
    const uint32_t j0 = (threadIdx.x & 63) * 4;
    const uint32_t j_step[4] = {j0 * LANE_STEP, (j0 + 1) * LANE_STEP, (j0 + 2) * LANE_STEP, (j0 + 3) * LANE_STEP};
    const uint32_t key = mix32(mix32(mix32(seed) + (uint32_t)__builtin_amdgcn_readfirstlane(e.step)) + (uint32_t)R.index);
    // a wave takes BLOCKS blocks, 4 apart: the workgroup's waves work on neighbouring blocks at a time
    const uint32_t blk0 = (uint32_t)(at.first / VCR_OPT_BLOCK) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t nblocks = (uint32_t)((R.numel + VCR_OPT_BLOCK - 1) / VCR_OPT_BLOCK);
#pragma unroll 1
    for (uint32_t i = 0; i < BLOCKS; ++i) {
        const uint32_t blk = blk0 + 4 * i;
        if (blk >= nblocks) break;
        const long long first = (long long)blk * VCR_OPT_BLOCK, have = R.numel - first;
        Block8<T> b;
        b.g = global(grad) + first;
        b.p = global((T*)R.p) + first;
        b.mst = MASTER ? global(R.master) + first : nullptr;
        b.mc = global((uint8_t*)R.m) + first;
        b.vc = global((uint8_t*)R.v) + first;
        b.whole = have >= VCR_OPT_BLOCK;
        b.n = b.whole ? 4 : have > j0 ? (int)min((long long)4, have - j0) : 0;
        Lane8 r = load_block<T, MASTER>(b, j0);
        GLOBAL uint8_t *ms = global(R.m_scale) + blk, *vs = global(R.v_scale) + blk;
        int sm = __builtin_amdgcn_readfirstlane(*ms), sv = __builtin_amdgcn_readfirstlane(*vs);
        const uint32_t bkey = mix32(key + blk);
        if (!b.whole || !block_fast(r, sm, sv, bkey, j_step, gs, e.coef, fast)) block_any(r, sm, sv, bkey, j_step, b.n, gs, e.coef);
        store_block<T, MASTER>(b, j0, r);
        if (j0 == 0) { *ms = (uint8_t)sm; *vs = (uint8_t)sv; }
    }
    leave<BLOCKS>(R, words, at, e.step);
}

// ---- codes -> values, values -> codes (to the nearest, ties to even) ------------------------------------------------------
// Elements per lane: what 16 bytes of output hold (295 M elements into bfloat16: 280 us, 6.3 TB/s, against 369 us with four each).
template <typename T> constexpr int decode_width() { return 16 / sizeof(T); }
template <typename T>
__global__ void __launch_bounds__(VCR_OPT_THREADS) decode_kernel(const VcrOptimTensor* __restrict__ tensors, const uint2* __restrict__ chunks,
                                                                 PairPack out, int t0) {
    constexpr int V = decode_width<T>();
    const Place at = place<V / 4>(chunks);
    const VcrOptimTensor& R = tensors[at.tensor];
    const long long off = at.first + threadIdx.x * V, left = R.numel - off;
    if (left <= 0 || !R.m_scale) return;
    GLOBAL T *mo = global((T*)out.a[at.tensor - t0]), *vo = global((T*)out.b[at.tensor - t0]);
    const GLOBAL uint8_t *mc = global((const uint8_t*)R.m) + off, *vc = global((const uint8_t*)R.v) + off;
    const int sm = global(R.m_scale)[off / VCR_OPT_BLOCK], sv = global(R.v_scale)[off / VCR_OPT_BLOCK];
    uint32_t cm[V / 4] = {}, cv[V / 4] = {};
    if (left >= V) {
        if constexpr (V == 8) {
            const u2b m = ldq<true, u2b>(mc), v = ldq<true, u2b>(vc);
            cm[0] = m.x; cm[1] = m.y; cv[0] = v.x; cv[1] = v.y;
        } else {
            cm[0] = ldq<true, u1a>(mc);
            cv[0] = ldq<true, u1a>(vc);
        }
    } else {
#pragma unroll
        for (int k = 0; k < V - 1; ++k)
            if (k < left) { cm[k / 4] |= (uint32_t)mc[k] << (8 * (k & 3)); cv[k / 4] |= (uint32_t)vc[k] << (8 * (k & 3)); }
    }
    Vec<V> m, v;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        m.x[k] = decode_m(cm[k / 4] >> (8 * (k & 3)) & 255u, sm);
        v.x[k] = decode_v(cv[k / 4] >> (8 * (k & 3)) & 255u, sv);
    }
    if (left >= V) {
        if (mo) storev<V, true>(mo + off, m);
        if (vo) storev<V, true>(vo + off, v);
    } else {
#pragma unroll
        for (int k = 0; k < V - 1; ++k)
            if (k < left) {
                if (mo) store1(mo + off + k, m.x[k]);
                if (vo) store1(vo + off + k, v.x[k]);
            }
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
// One block of 256 values, four of them 64 apart in each lane, as codes and exponents.
__device__ __forceinline__ void encode_block(const float (&m)[4], const float (&v)[4], long long blk, uint32_t lane, long long numel,
                                             GLOBAL uint8_t* mc, GLOBAL uint8_t* vc, GLOBAL uint8_t* ms, GLOBAL uint8_t* vs) {
    uint32_t mb = 0, vb = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) { mb = max(mb, finite_bits(m[k])); vb = max(vb, finite_bits(v[k])); }
    const int nm = scale_of(rows_max(row_max(mb))), nv = scale_of(rows_max(row_max(vb)));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const long long i = blk * VCR_OPT_BLOCK + lane + 64 * k;
        if (i < numel) { mc[i] = (uint8_t)nearest_m(m[k], nm); vc[i] = (uint8_t)nearest_v(v[k], nv); }
    }
    if (lane == 0) { ms[blk] = (uint8_t)nm; vs[blk] = (uint8_t)nv; }
}
__global__ void __launch_bounds__(256) encode_kernel(const VcrOptimTensor* __restrict__ tensors, const uint2* __restrict__ chunks,
                                                     PairPack in, int t0) {
    const uint2 cw = chunks[blockIdx.x];
    const VcrOptimTensor& R = tensors[cw.x];
    if (!R.m_scale) return;
    const GLOBAL float *mi = global((const float*)in.a[cw.x - t0]), *vi = global((const float*)in.b[cw.x - t0]);
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t b = threadIdx.x >> 6; b < VCR_OPT_CHUNK / VCR_OPT_BLOCK; b += 4) {
        const long long blk = (long long)cw.y * (VCR_OPT_CHUNK / VCR_OPT_BLOCK) + b, first = blk * VCR_OPT_BLOCK + lane;
        if (blk * VCR_OPT_BLOCK >= R.numel) break;
        float m[4], v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const long long i = first + 64 * k;
            m[k] = i < R.numel ? mi[i] : 0.f;
            v[k] = i < R.numel ? vi[i] : 0.f;
        }
        encode_block(m, v, blk, lane, R.numel, global((uint8_t*)R.m), global((uint8_t*)R.v), global(R.m_scale), global(R.v_scale));
    }
}

// Rows of 8-bit moments in another order: row r of the output is row index[r] of the input, zeros where that is no row.  One wave per
// block of the output, whose exponents are formed anew from the values that land in it; four elements per lane, gathered one by one
// (a row is shorter than a block, and begins anywhere).  Read and written are codes: expanded to fp32 and back the moments would
// take 16 bytes a parameter on the way instead of 4, more than a caller who chose 8 bits has.
__global__ void __launch_bounds__(256) rows8_kernel(VcrRows8 A, long long rows_in, long long numel, const int32_t* __restrict__ index) {
    const long long blk = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (blk * VCR_OPT_BLOCK >= numel) return;
    const uint32_t lane = threadIdx.x & 63;
    const GLOBAL uint8_t *mc = global(A.m), *vc = global(A.v), *ms = global(A.m_scale), *vs = global(A.v_scale);
    float m[4], v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const long long i = blk * VCR_OPT_BLOCK + lane + 64 * k;
        m[k] = v[k] = 0.f;
        if (i >= numel) continue;
        const long long row = i / A.width, from = global(index)[row];
        if (from < 0 || from >= rows_in) continue;
        const long long e = from * A.width + (i - row * A.width);
        m[k] = decode_m(mc[e], ms[e / VCR_OPT_BLOCK]);
        v[k] = decode_v(vc[e], vs[e / VCR_OPT_BLOCK]);
    }
    encode_block(m, v, blk, lane, numel, global(A.m_out), global(A.v_out), global(A.m_scale_out), global(A.v_scale_out));
}

// ---- host side ---------------------------------------------------------------------------------------------------------
inline int64_t chunks_of(int64_t numel, int64_t chunk) { return numel / chunk + (numel % chunk != 0); }          // (no overflow)
// entries of a plan: a tensor without elements has one too, for its counter
inline int64_t entries_of(int64_t numel) { return numel > 0 ? chunks_of(numel, VCR_OPT_CHUNK) : 1; }
inline size_t plan_head(int n) { return vcr_align(sizeof(VcrOptimTensor) * (size_t)n); }
inline size_t plan_words(int n, int64_t chunks) { return vcr_align(plan_head(n) + sizeof(uint2) * (size_t)chunks); }
inline uint32_t tickets_of(int64_t chunks) { return chunks > TICKET_FLAT ? 1 + TICKET_GROUPS : 1; }
inline const uint2* plan_chunks(const void* plan, int n) { return (const uint2*)((const char*)plan + plan_head(n)); }

// checks that the calls on a plan share; returns the number of chunks, -1 with an error set
int64_t plan_check(const char* who, const void* plan, int n, const int64_t* numel) {
    if (!plan || !numel || n < 1) { vcr_set_error("%s: plan or numel is missing", who); return -1; }
    int64_t total = 0;
    for (int k = 0; k < n; ++k) {
        if (numel[k] < 0) { vcr_set_error("%s: tensor %d has numel %lld", who, k, (long long)numel[k]); return -1; }
        if (entries_of(numel[k]) > VCR_OPT_LAUNCH_CHUNKS) { vcr_set_error("%s: tensor %d with %lld elements is too large", who, k, (long long)numel[k]); return -1; }
        total += entries_of(numel[k]);
    }
    if (total > 0x0FFFFFFF) { vcr_set_error("%s: %lld chunks", who, (long long)total); return -1; }
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
            if (start + c > NORM_LAUNCH_CHUNKS) break;
            pk.g[used] = tensors[k];
            pk.n[used] = numel[k];
            start += c;
            pk.start[++used] = (uint32_t)start;
        }
        if (used == 0) break;
        if (launch(pk, used, (uint32_t)start)) return 1;
    }
    return 0;
}

int list_check(const char* who, int n, const void* const* tensors, const int64_t* numel, const int32_t* types) {
    if (n < 0 || (n > 0 && (!tensors || !numel || !types))) { vcr_set_error("%s: the list of tensors is missing", who); return 1; }
    for (int k = 0; k < n; ++k) {
        if (numel[k] < 0 || (numel[k] > 0 && !tensors[k]) || types[k] < 0 || types[k] > VCR_F16) {
            vcr_set_error("%s: tensor %d has numel %lld, pointer %p, type %d", who, k, (long long)numel[k], tensors[k], types[k]);
            return 1;
        }
        if (chunks_of(numel[k], NORM_CHUNK) > NORM_LAUNCH_CHUNKS) { vcr_set_error("%s: tensor %d with %lld elements is too large", who, k, (long long)numel[k]); return 1; }
    }
    return 0;
}

}  // namespace

extern "C" size_t vcr_optim_plan_bytes(int ntensors, const int64_t* numel) {
    if (ntensors < 1 || !numel) return 0;
    int64_t total = 0;
    size_t tickets = 0;
    for (int k = 0; k < ntensors; ++k) {
        const int64_t nc = entries_of(numel[k]);
        if (nc > VCR_OPT_LAUNCH_CHUNKS) return 0;          // (vcr_optim_plan says why)
        total += nc;
        tickets += tickets_of(nc);
    }
    return plan_words(ntensors, total) + tickets * TICKET_STRIDE * sizeof(uint32_t);
}

extern "C" int vcr_optim_plan(int ntensors, const VcrOptimTensor* tensors, void* host_plan, size_t bytes) {
    if (ntensors < 1 || !tensors || !host_plan) { vcr_set_error("vcr_optim_plan: tensors or plan is missing"); return 1; }
    int64_t total = 0;
    size_t tickets = 0;
    for (int k = 0; k < ntensors; ++k) {
        const VcrOptimTensor& t = tensors[k];
        if (t.numel < 0 || !t.step || (t.numel > 0 && (!t.p || !t.m || !t.v)) || (!t.m_scale != !t.v_scale)) {
            vcr_set_error("vcr_optim_plan: tensor %d has numel %lld and a pointer missing", k, (long long)t.numel);
            return 1;
        }
        if (entries_of(t.numel) > VCR_OPT_LAUNCH_CHUNKS) { vcr_set_error("vcr_optim_plan: tensor %d with %lld elements is too large", k, (long long)t.numel); return 1; }
        total += entries_of(t.numel);
        tickets += tickets_of(entries_of(t.numel));
    }
    const size_t words = plan_words(ntensors, total), need = words + tickets * TICKET_STRIDE * sizeof(uint32_t);
    if (total > 0x0FFFFFFF || tickets > 0x7FFFFFFF || bytes < need) { vcr_set_error("vcr_optim_plan: %zu bytes for %lld chunks", bytes, (long long)total); return 1; }
    VcrOptimTensor* out = (VcrOptimTensor*)host_plan;
    uint2* c = (uint2*)((char*)host_plan + plan_head(ntensors));
    int32_t word = 0;
    for (int k = 0; k < ntensors; ++k) {
        const uint32_t nc = (uint32_t)entries_of(tensors[k].numel);
        out[k] = tensors[k];
        out[k].words = word;
        word += (int32_t)tickets_of(nc);
        for (uint32_t i = 0; i < nc; ++i) *c++ = make_uint2((uint32_t)k, i);
    }
    memset((char*)host_plan + words, 0, need - words);
    return 0;
}

extern "C" int vcr_adamw_step(const VcrAdamWStep* args, void* stream) {
    if (!args) { vcr_set_error("vcr_adamw_step: args is NULL"); return 1; }
    const VcrAdamWStep& a = *args;
    if (a.ntensors == 0) return 0;
    const int64_t nall = plan_check("vcr_adamw_step", a.plan, a.ntensors, a.numel);
    if (nall < 0) return 1;
    if (!a.grads || !a.groups || !a.group_of || a.ngroups < 1 || a.param_type < 0 || a.param_type > VCR_F16 ||
        (a.state_bits != 32 && a.state_bits != 8) || (a.masters && a.param_type == VCR_F32)) {
        vcr_set_error("vcr_adamw_step: inconsistent arguments");
        return 1;
    }
    for (int k = 0; k < a.ngroups; ++k) {
        const VcrOptimGroup& g = a.groups[k];
        if (!(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0 && (g.eps == 0.0 || g.eps >= 0x1p-126))) {
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
    uint32_t* words = (uint32_t*)((char*)a.plan + plan_words(a.ntensors, nall));
    const Clip* clip = (const Clip*)a.clip;
    for (int t0 = 0, t1 = 0; t0 < a.ntensors; t0 = t1) {
        StepPack pk = {};
        int64_t nchunks = 0;
        bool any = false;
        const int g0 = a.group_of[t0];
        for (; t1 < a.ntensors && t1 - t0 < VCR_OPT_TENSORS && a.group_of[t1] - g0 < VCR_OPT_GROUPS; ++t1) {
            const int64_t c = entries_of(a.numel[t1]);
            if (nchunks + c > VCR_OPT_LAUNCH_CHUNKS) break;
            pk.g[t1 - t0] = a.grads[t1];
            nchunks += c;
            any |= a.grads[t1] != nullptr;
        }
        for (int k = g0; k <= a.group_of[t1 - 1]; ++k) {
            const VcrOptimGroup& g = a.groups[k];
            pk.group[k - g0] = {g.lr, g.weight_decay, log(g.beta1), log(g.beta2), g.lr_dev, (float)g.eps,
                                (float)g.beta1, (float)(1.0 - g.beta1), (float)g.beta2, (float)(1.0 - g.beta2), 0};
        }
        if (any) {
            const dim3 block(VCR_OPT_THREADS);
            const float gs = (float)a.grad_scale;
#define LAUNCH32(T, M) hipLaunchKernelGGL((adamw_kernel<T, M>), dim3((uint32_t)nchunks * parts<1>()), block, 0, st, tensors, chunks, words, clip, gs, pk, t0, g0)
#define LAUNCH8(T, M) hipLaunchKernelGGL((adamw8_kernel<T, M>), dim3((uint32_t)nchunks * parts<blocks8<T, M>()>()), block, 0, st, tensors, chunks, words, clip, gs, pk, t0, g0, a.seed)
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

static int pairs_call(const char* who, int n, const void* plan, const int64_t* numel, const void* const* a, const void* const* b,
                      int type, bool encode, hipStream_t st) {
    if (n == 0) return 0;
    if (plan_check(who, plan, n, numel) < 0) return 1;
    if (!a || !b || type < 0 || type > VCR_F16) { vcr_set_error("%s: inconsistent arguments", who); return 1; }
    const VcrOptimTensor* tensors = (const VcrOptimTensor*)plan;
    const uint2* chunks = plan_chunks(plan, n);
    for (int t0 = 0, t1 = 0; t0 < n; t0 = t1) {
        PairPack pk = {};
        int64_t nchunks = 0;
        for (; t1 < n && t1 - t0 < VCR_OPT_PAIRS; ++t1) {
            const int64_t c = entries_of(numel[t1]);
            if (nchunks + c > VCR_OPT_LAUNCH_CHUNKS) break;
            pk.a[t1 - t0] = a[t1];
            pk.b[t1 - t0] = b[t1];
            if (encode && numel[t1] > 0 && (!a[t1] || !b[t1])) { vcr_set_error("%s: values of tensor %d are missing", who, t1); return 1; }
            nchunks += c;
        }
        if (nchunks > 0) {
            const uint32_t per = encode ? 1 : type == VCR_F32 ? parts<decode_width<float>() / 4>() : parts<decode_width<__half>() / 4>();
            const dim3 grid((uint32_t)nchunks * per), block(VCR_OPT_THREADS);
            if (encode) hipLaunchKernelGGL(encode_kernel, grid, block, 0, st, tensors, chunks, pk, t0);
            else if (type == VCR_F32) hipLaunchKernelGGL(decode_kernel<float>, grid, block, 0, st, tensors, chunks, pk, t0);
            else if (type == VCR_BF16) hipLaunchKernelGGL(decode_kernel<__hip_bfloat16>, grid, block, 0, st, tensors, chunks, pk, t0);
            else hipLaunchKernelGGL(decode_kernel<__half>, grid, block, 0, st, tensors, chunks, pk, t0);
        }
        chunks += nchunks;
    }
    VCR_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int vcr_moments8_decode(int ntensors, const void* plan, const int64_t* numel, void* const* exp_avg,
                                   void* const* exp_avg_sq, int type, void* stream) {
    return pairs_call("vcr_moments8_decode", ntensors, plan, numel, exp_avg, exp_avg_sq, type, false, (hipStream_t)stream);
}
extern "C" int vcr_moments8_encode(int ntensors, const void* plan, const int64_t* numel, const float* const* exp_avg,
                                   const float* const* exp_avg_sq, void* stream) {
    return pairs_call("vcr_moments8_encode", ntensors, plan, numel, (const void* const*)exp_avg, (const void* const*)exp_avg_sq, VCR_F32,
                      true, (hipStream_t)stream);
}

extern "C" int vcr_moments8_rows(int narrays, const VcrRows8* arrays, int64_t rows_in, int64_t rows_out, const int32_t* index, void* stream) {
    if (narrays < 0 || (narrays > 0 && !arrays) || rows_in < 0 || rows_out < 0 || (rows_out > 0 && !index)) {
        vcr_set_error("vcr_moments8_rows: inconsistent arguments");
        return 1;
    }
    const int64_t most = (int64_t)VCR_OPT_LAUNCH_CHUNKS * VCR_OPT_CHUNK;
    for (int k = 0; k < narrays; ++k) {
        const VcrRows8& a = arrays[k];
        if (a.width < 1 || rows_in > most / a.width || rows_out > most / a.width) {
            vcr_set_error("vcr_moments8_rows: array %d has width %d, %lld rows -> %lld", k, a.width, (long long)rows_in, (long long)rows_out);
            return 1;
        }
        if ((rows_in > 0 && (!a.m || !a.v || !a.m_scale || !a.v_scale)) || (rows_out > 0 && (!a.m_out || !a.v_out || !a.m_scale_out || !a.v_scale_out))) {
            vcr_set_error("vcr_moments8_rows: array %d has a pointer missing", k);
            return 1;
        }
    }
    if (rows_out == 0) return 0;
    for (int k = 0; k < narrays; ++k) {
        const int64_t numel = rows_out * arrays[k].width;
        hipLaunchKernelGGL(rows8_kernel, dim3((uint32_t)chunks_of(numel, 4 * VCR_OPT_BLOCK)), dim3(256), 0, (hipStream_t)stream, arrays[k], (long long)rows_in,
                           (long long)numel, index);
    }
    VCR_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int vcr_grad_norm_partials(int ntensors, const int64_t* numel) {
    if (ntensors < 1 || !numel) return 1;
    int64_t chunks = 0;
    for (int k = 0; k < ntensors; ++k) {
        const int64_t c = numel[k] > 0 ? chunks_of(numel[k], NORM_CHUNK) : 0;
        if (c <= NORM_LAUNCH_CHUNKS) chunks += c;          // (a larger one is refused by vcr_grad_norm)
    }
    const int64_t packs = ntensors / VCR_OPT_NORM_TENSORS + 3 + chunks / 0x40000000;     // (a pack ends with its type)
    const int64_t most = packs * VCR_OPT_NORM_BLOCKS;
    return (int)(chunks < most ? chunks + 1 : most);
}

extern "C" int vcr_grad_norm(int ntensors, const void* const* tensors, const int64_t* numel, const int32_t* types, double* partials,
                             int capacity, double grad_scale, double max_norm, int read_again, float* norm, void* clip, void* stream) {
    if (list_check("vcr_grad_norm", ntensors, tensors, numel, types)) return 1;
    if (!partials || (!norm && !clip)) { vcr_set_error("vcr_grad_norm: partials or norm is NULL"); return 1; }
    if (clip && !(max_norm > 0.0)) { vcr_set_error("vcr_grad_norm: max_norm is %g", max_norm); return 1; }
    hipStream_t st = (hipStream_t)stream;
    const Finish f{grad_scale, max_norm, norm, (Clip*)clip};
    int used_partials = 0, types_seen = 0;
    int64_t all = 0, listed = 0;
    for (int k = 0; k < ntensors; ++k)
        if (numel[k] > 0) { types_seen |= 1 << types[k]; all += chunks_of(numel[k], NORM_CHUNK); ++listed; }
    const bool one = all <= VCR_OPT_NORM_ONE && listed <= VCR_OPT_NORM_TENSORS && (types_seen & (types_seen - 1)) == 0 && all > 0;
    for (int type = VCR_F32; type <= VCR_F16; ++type) {
        const int rc = each_norm_pack(ntensors, tensors, numel, types, type, [&](const NormPack& pk, int used, uint32_t chunks) {
            const int blocks = one ? 1 : chunks < VCR_OPT_NORM_BLOCKS ? (int)chunks : VCR_OPT_NORM_BLOCKS;
            if (used_partials + blocks > capacity) { vcr_set_error("vcr_grad_norm: room for %d partial sums is too little", capacity); return 1; }
            double* out = partials + used_partials;
#define LAUNCH(T, NT, ONE) hipLaunchKernelGGL((norm_kernel<T, NT, ONE>), dim3(blocks), dim3(norm_threads<T, NT, ONE>()), 0, st, pk, used, NORM_CHUNK, out, f)
#define LAUNCH_ANY(T) do { if (one) LAUNCH(T, false, true); else if (read_again) LAUNCH(T, false, false); else LAUNCH(T, true, false); } while (0)
            if (type == VCR_F32) LAUNCH_ANY(float);
            else if (type == VCR_BF16) LAUNCH_ANY(__hip_bfloat16);
            else LAUNCH_ANY(__half);
#undef LAUNCH_ANY
#undef LAUNCH
            used_partials += blocks;
            return 0;
        });
        if (rc) return 1;
    }
    if (!one) hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(256), 0, st, partials, used_partials, f);
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
