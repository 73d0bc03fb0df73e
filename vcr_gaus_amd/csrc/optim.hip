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
#define VCR_OPT_TENSORS 400        // tensors per launch: their gradient pointers travel in the kernel arguments (4 KB)
#define VCR_OPT_GROUPS 48          // hyper-parameter groups per launch of the begin kernel
#define VCR_OPT_NORM_TENSORS 192   // tensors per launch of the norm kernel
#define VCR_OPT_PAIRS 200          // tensors per launch of the code <-> value kernels
#define VCR_OPT_NORM_BLOCKS 1024

struct GradPack { const void* g[VCR_OPT_TENSORS]; };
struct GroupPack { VcrOptimGroup g[VCR_OPT_GROUPS]; };
struct LivePack { uint32_t w[(VCR_OPT_TENSORS + 31) / 32]; };
struct PairPack { const void* a[VCR_OPT_PAIRS]; const void* b[VCR_OPT_PAIRS]; };
struct NormPack { const void* g[VCR_OPT_NORM_TENSORS]; long long n[VCR_OPT_NORM_TENSORS]; uint32_t start[VCR_OPT_NORM_TENSORS + 1]; };

// per-step factors of one tensor, written by the begin kernel
struct Coef { float decay, step_size, inv_sqrt_bc2, eps, b1, omb1, b2, omb2; };
struct Head { float gscale; int skip; uint32_t pad[6]; };      // in front of the Coef records
static_assert(sizeof(Coef) == 32 && sizeof(Head) == 32, "the factors of a step are 32-byte records");

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __hip_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load1(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(__hip_bfloat16* p, float x) { *p = __float2bfloat16(x); }
__device__ __forceinline__ void store1(__half* p, float x) { *p = __float2half(x); }

__device__ __forceinline__ void moments_one(float& m, float& v, float g, const Coef& c) {
#pragma clang fp contract(off)
    m = m * c.b1 + g * c.omb1;
    v = v * c.b2 + (g * g) * c.omb2;
}
__device__ __forceinline__ float param_one(float p, float m, float v, const Coef& c) {
    return p * c.decay - c.step_size * (m / (sqrtf(v) * c.inv_sqrt_bc2 + c.eps));
}

// 32-bit mix (constants found by a search for even avalanche over counters and random words)
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x582C52E9u;
    x = (x ^ (x >> 15)) * 0x1B156CA9u;
    return x ^ (x >> 16);
}
// the random word of an element: `key` = mix32 of (seed, step, tensor, block); one more multiplication spreads the lane
__device__ __forceinline__ uint32_t element_word(uint32_t key, uint32_t j) {
    uint32_t x = key ^ (j * 0x9E3779B1u);
    x = (x ^ (x >> 16)) * 0x582C52E9u;
    return x ^ (x >> 15);
}

#define M_TOP 14
#define V_TOP 30
__device__ __forceinline__ float decode_m(uint32_t c, int s) {
    const float x = ldexpf(__uint_as_float((c & 0x7Fu) << 20), s - M_TOP);
    return __uint_as_float(((c & 0x7Fu) == 0x7Fu ? 0x7FC00000u : __float_as_uint(x)) | ((c & 0x80u) << 24));
}
__device__ __forceinline__ float decode_v(uint32_t c, int s) {
    return c == 0xFFu ? __uint_as_float(0x7FC00000u) : ldexpf(__uint_as_float(c << 20), s - V_TOP);
}
__device__ __forceinline__ uint32_t encode_m(float m, int s, uint32_t r) {
    const uint32_t b = __float_as_uint(m), a = b & 0x7FFFFFFFu;
    const uint32_t c = a >= 0x7F800000u ? 0x7Fu : (__float_as_uint(ldexpf(__uint_as_float(a), M_TOP - s)) + r) >> 20;
    return c | (b >> 24 & 0x80u);
}
__device__ __forceinline__ uint32_t encode_v(float v, int s, uint32_t r) {
    const uint32_t a = __float_as_uint(v) & 0x7FFFFFFFu;
    if (a >= 0x7F800000u) return 0xFFu;
    const uint32_t c = (__float_as_uint(ldexpf(__uint_as_float(a), V_TOP - s)) + r) >> 20;
    return c == 0u && a != 0u ? 1u : c;
}
// largest finite magnitude as float bits (0 for what is not finite)
__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t a = __float_as_uint(x) & 0x7FFFFFFFu;
    return a >= 0x7F800000u ? 0u : a;
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

template <typename T>
__global__ void __launch_bounds__(256) norm_kernel(NormPack pk, int n, uint32_t chunk, double* __restrict__ partials) {
    __shared__ double lds[4];
    double sum = 0.0;
    for (uint32_t c = blockIdx.x; c < pk.start[n]; c += gridDim.x) {
        int lo = 0, hi = n - 1;                    // the tensor whose chunks hold c
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pk.start[mid] <= c) lo = mid; else hi = mid - 1;
        }
        const T* g = (const T*)pk.g[lo];
        const long long off = (long long)(c - pk.start[lo]) * chunk;
        const long long left = pk.n[lo] - off;
        const uint32_t cnt = left < (long long)chunk ? (uint32_t)left : chunk;
        g += off;
        for (uint32_t i = threadIdx.x; i < cnt; i += 256) { const double x = (double)load1(g + i); sum += x * x; }
    }
    sum = block_sum(sum, lds);
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

__device__ __forceinline__ double sum_partials(const double* __restrict__ partials, int n, double* lds) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += partials[i];
    return block_sum(s, lds);
}

__global__ void __launch_bounds__(256) norm_final_kernel(const double* __restrict__ partials, int n, double scale,
                                                         float* __restrict__ out) {
    __shared__ double lds[4];
    const double s = sum_partials(partials, n, lds);
    if (threadIdx.x == 0) *out = (float)(sqrt(s) * scale);
}

// g *= min(1, max_norm / (norm + 1e-6)); a norm that is not finite leaves NaN or zero as the formula says
template <typename T>
__global__ void __launch_bounds__(256) scale_kernel(NormPack pk, int n, uint32_t chunk, const float* __restrict__ norm, double max_norm) {
    const double q = max_norm / ((double)*norm + 1e-6);
    const float f = q > 1.0 ? 1.f : (float)q;
    if (f == 1.f) return;
    for (uint32_t c = blockIdx.x; c < pk.start[n]; c += gridDim.x) {
        int lo = 0, hi = n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pk.start[mid] <= c) lo = mid; else hi = mid - 1;
        }
        T* g = (T*)pk.g[lo];
        const long long off = (long long)(c - pk.start[lo]) * chunk;
        const long long left = pk.n[lo] - off;
        const uint32_t cnt = left < (long long)chunk ? (uint32_t)left : chunk;
        g += off;
        for (uint32_t i = threadIdx.x; i < cnt; i += 256) store1(g + i, load1(g + i) * f);
    }
}

// ---- begin of a step: clipping, step counters, bias corrections ---------------------------------------------------------
// One workgroup.  Advances the counter of every stepped tensor and writes its factors; a norm that is not finite sets `skip`
// (no counter moves, the update kernels return at once).
__global__ void __launch_bounds__(256) begin_kernel(const VcrOptimTensor* __restrict__ tensors, int t0, int nt, LivePack live,
                                                    GroupPack groups, int g0, int ng, const double* __restrict__ partials,
                                                    int npartials, double grad_scale, double max_norm, float* __restrict__ norm_out,
                                                    Head* __restrict__ head, Coef* __restrict__ coef) {
    __shared__ double lds[4];
    float gscale = (float)grad_scale;
    int skip = 0;
    if (npartials > 0) {
        const double norm = sqrt(sum_partials(partials, npartials, lds)) * fabs(grad_scale);
        const double q = max_norm / ((double)(float)norm + 1e-6);
        skip = !(norm <= 3.0e38);
        if (q < 1.0) gscale = (float)(grad_scale * q);
        if (threadIdx.x == 0 && norm_out) *norm_out = (float)norm;
    }
    if (threadIdx.x == 0) { head->gscale = gscale; head->skip = skip; }
    if (skip) return;
    for (int k = threadIdx.x; k < nt; k += 256) {
        if (!(live.w[k >> 5] >> (k & 31) & 1u)) continue;
        const VcrOptimTensor& T = tensors[t0 + k];
        const int gi = T.group - g0;
        if (gi < 0 || gi >= ng) continue;
        const VcrOptimGroup& G = groups.g[gi];
        const int t = *T.step + 1;
        *T.step = t;
        const double lr = G.lr_dev ? (double)*G.lr_dev : G.lr;
        const double bc1 = -expm1((double)t * log(G.beta1)), bc2 = -expm1((double)t * log(G.beta2));
        Coef c;
        c.decay = (float)(1.0 - lr * G.weight_decay);
        c.step_size = (float)(lr / bc1);
        c.inv_sqrt_bc2 = (float)(1.0 / sqrt(bc2));
        c.eps = (float)G.eps;
        c.b1 = (float)G.beta1; c.omb1 = (float)(1.0 - G.beta1);
        c.b2 = (float)G.beta2; c.omb2 = (float)(1.0 - G.beta2);
        coef[t0 + k] = c;
    }
}

// ---- update, moments in 32 bits --------------------------------------------------------------------------------------
template <typename T, bool MASTER>
__global__ void __launch_bounds__(256) adamw_kernel(const VcrOptimTensor* __restrict__ tensors, const uint2* __restrict__ chunks,
                                                    uint32_t chunk, const Head* __restrict__ head, const Coef* __restrict__ coef,
                                                    GradPack grads, int t0) {
    const uint2 cw = chunks[blockIdx.x];
    const T* g = (const T*)grads.g[cw.x - t0];
    if (!g || head->skip) return;
    const VcrOptimTensor& R = tensors[cw.x];
    const Coef c = coef[cw.x];
    const float gs = head->gscale;
    const long long off = (long long)cw.y * chunk;
    const long long left = R.numel - off;
    const uint32_t cnt = left < (long long)chunk ? (uint32_t)left : chunk;
    T* p = (T*)R.p + off;
    float* mst = MASTER ? R.master + off : nullptr;
    float *m = (float*)R.m + off, *v = (float*)R.v + off;
    g += off;
    for (uint32_t i = threadIdx.x; i < cnt; i += 256) {
        float mm = m[i], vv = v[i];
        moments_one(mm, vv, load1(g + i) * gs, c);
        const float x = param_one(MASTER ? mst[i] : load1(p + i), mm, vv, c);
        m[i] = mm; v[i] = vv;
        if (MASTER) mst[i] = x;
        store1(p + i, x);
    }
}

// ---- update, moments in 8 bits: one wave per block of 256, four consecutive elements per lane ---------------------------
template <typename T, bool MASTER>
__global__ void __launch_bounds__(256) adamw8_kernel(const VcrOptimTensor* __restrict__ tensors, const uint2* __restrict__ chunks,
                                                     uint32_t chunk, const Head* __restrict__ head, const Coef* __restrict__ coef,
                                                     GradPack grads, int t0, uint32_t seed) {
    const uint2 cw = chunks[blockIdx.x];
    const T* g = (const T*)grads.g[cw.x - t0];
    if (!g || head->skip) return;
    const VcrOptimTensor& R = tensors[cw.x];
    const Coef c = coef[cw.x];
    const float gs = head->gscale;
    const long long off = (long long)cw.y * chunk;
    const long long left = R.numel - off;
    const uint32_t cnt = left < (long long)chunk ? (uint32_t)left : chunk;
    T* p = (T*)R.p + off;
    float* mst = MASTER ? R.master + off : nullptr;
    uint8_t *mc = (uint8_t*)R.m + off, *vc = (uint8_t*)R.v + off;
    g += off;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t key = mix32(mix32(mix32(seed) + (uint32_t)*R.step) + (uint32_t)R.index);
    for (uint32_t b = threadIdx.x >> 6; b * VCR_OPT_BLOCK < cnt; b += 4) {
        const long long blk = off / VCR_OPT_BLOCK + b;
        const uint32_t j0 = lane * 4, base = b * VCR_OPT_BLOCK + j0;
        const int sm = R.m_scale[blk], sv = R.v_scale[blk];
        float mm[4], vv[4];
        uint32_t mb = 0, vb = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            mm[k] = vv[k] = 0.f;
            if (base + k < cnt) {
                const uint32_t i = base + k;
                mm[k] = decode_m(mc[i], sm);
                vv[k] = decode_v(vc[i], sv);
                moments_one(mm[k], vv[k], load1(g + i) * gs, c);
                const float x = param_one(MASTER ? mst[i] : load1(p + i), mm[k], vv[k], c);
                if (MASTER) mst[i] = x;
                store1(p + i, x);
                mb = max(mb, finite_bits(mm[k]));
                vb = max(vb, finite_bits(vv[k]));
            }
        }
        const int nm = scale_of(wave_max(mb)), nv = scale_of(wave_max(vb));
        const uint32_t bkey = mix32(key + (uint32_t)blk);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (base + k < cnt) {
                const uint32_t x = element_word(bkey, j0 + k);
                mc[base + k] = (uint8_t)encode_m(mm[k], nm, (x >> 16) * 16u + 8u);
                vc[base + k] = (uint8_t)encode_v(vv[k], nv, (x & 65535u) * 16u + 8u);
            }
        }
        if (lane == 0) { R.m_scale[blk] = (uint8_t)nm; R.v_scale[blk] = (uint8_t)nv; }
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

template <typename F>
int each_norm_pack(int n, const void* const* tensors, const int64_t* numel, uint32_t chunk, F launch) {
    int k = 0;
    while (k < n) {
        NormPack pk;
        int used = 0;
        uint64_t start = 0;
        pk.start[0] = 0;
        for (; k < n && used < VCR_OPT_NORM_TENSORS; ++k) {
            if (numel[k] == 0) continue;
            const uint64_t c = (uint64_t)chunks_of(numel[k], chunk);
            if (start + c > 0x7FFFFFFFull) break;
            pk.g[used] = tensors[k];
            pk.n[used] = numel[k];
            start += c;
            pk.start[++used] = (uint32_t)start;
        }
        if (used == 0) {
            if (k < n) { vcr_set_error("tensor %d is too large", k); return 1; }
            break;
        }
        if (launch(pk, used, (uint32_t)start)) return 1;
    }
    return 0;
}

int list_check(const char* who, int n, const void* const* tensors, const int64_t* numel, int type) {
    if (n < 0 || type < 0 || type > VCR_F16 || (n > 0 && (!tensors || !numel))) { vcr_set_error("%s: bad list of tensors or type %d", who, type); return 1; }
    for (int k = 0; k < n; ++k)
        if (numel[k] < 0 || (numel[k] > 0 && !tensors[k])) { vcr_set_error("%s: tensor %d has numel %lld and pointer %p", who, k, (long long)numel[k], tensors[k]); return 1; }
    return 0;
}

#define NORM_CHUNK 16384

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
        if (t.numel < 0 || !t.step || (t.numel > 0 && (!t.p || !t.m || !t.v)) || (!t.m_scale != !t.v_scale)) {
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

extern "C" size_t vcr_adamw_work_bytes(int ntensors) { return ntensors < 1 ? 0 : sizeof(Head) + sizeof(Coef) * (size_t)ntensors; }

extern "C" int vcr_adamw_step(const VcrAdamWStep* args, void* stream) {
    if (!args) { vcr_set_error("vcr_adamw_step: args is NULL"); return 1; }
    const VcrAdamWStep& a = *args;
    if (a.ntensors == 0) return 0;
    if (plan_check("vcr_adamw_step", a.plan, a.ntensors, a.numel, a.chunk) < 0) return 1;
    if (!a.grads || !a.groups || a.ngroups < 1 || !a.work || a.param_type < 0 || a.param_type > VCR_F16 ||
        (a.state_bits != 32 && a.state_bits != 8) || (a.npartials > 0 && !a.partials) || a.npartials < 0 ||
        (a.masters && a.param_type == VCR_F32)) {
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
    hipStream_t st = (hipStream_t)stream;
    const VcrOptimTensor* tensors = (const VcrOptimTensor*)a.plan;
    const uint2* chunks = plan_chunks(a.plan, a.ntensors);
    Head* head = (Head*)a.work;
    Coef* coef = (Coef*)(head + 1);
    for (int t0 = 0; t0 < a.ntensors; t0 += VCR_OPT_TENSORS) {
        const int nt = a.ntensors - t0 < VCR_OPT_TENSORS ? a.ntensors - t0 : VCR_OPT_TENSORS;
        LivePack live = {};
        GradPack gp;
        int64_t nchunks = 0;
        for (int k = 0; k < nt; ++k) {
            gp.g[k] = a.grads[t0 + k];
            if (gp.g[k]) live.w[k >> 5] |= 1u << (k & 31);
            nchunks += chunks_of(a.numel[t0 + k], a.chunk);
        }
        for (int k = nt; k < VCR_OPT_TENSORS; ++k) gp.g[k] = nullptr;
        for (int g0 = 0; g0 < a.ngroups; g0 += VCR_OPT_GROUPS) {
            GroupPack pk = {};
            const int ng = a.ngroups - g0 < VCR_OPT_GROUPS ? a.ngroups - g0 : VCR_OPT_GROUPS;
            for (int k = 0; k < ng; ++k) pk.g[k] = a.groups[g0 + k];
            hipLaunchKernelGGL(begin_kernel, dim3(1), dim3(256), 0, st, tensors, t0, nt, live, pk, g0, ng, a.partials, a.npartials,
                               a.grad_scale, a.max_norm, a.norm_out, head, coef);
        }
        if (nchunks > 0) {
            const dim3 grid((uint32_t)nchunks), block(256);
#define LAUNCH32(T, M) hipLaunchKernelGGL((adamw_kernel<T, M>), grid, block, 0, st, tensors, chunks, (uint32_t)a.chunk, head, coef, gp, t0)
#define LAUNCH8(T, M) hipLaunchKernelGGL((adamw8_kernel<T, M>), grid, block, 0, st, tensors, chunks, (uint32_t)a.chunk, head, coef, gp, t0, a.seed)
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
    int64_t launches = 0, chunks = 0;
    if (ntensors < 0 || (ntensors > 0 && !numel)) return 0;
    for (int k = 0; k < ntensors; ++k) chunks += numel[k] > 0 ? chunks_of(numel[k], NORM_CHUNK) : 0;
    launches = (ntensors + VCR_OPT_NORM_TENSORS - 1) / VCR_OPT_NORM_TENSORS + chunks / 0x40000000 + 1;
    const int64_t most = launches * VCR_OPT_NORM_BLOCKS;
    return (int)(chunks < most ? chunks : most);
}

extern "C" int vcr_grad_norm_accumulate(int ntensors, const void* const* tensors, const int64_t* numel, int type, double* partials,
                                        int capacity, int* npartials, void* stream) {
    if (list_check("vcr_grad_norm_accumulate", ntensors, tensors, numel, type)) return 1;
    if (!npartials || *npartials < 0 || !partials) { vcr_set_error("vcr_grad_norm_accumulate: partials is NULL"); return 1; }
    const int rc = each_norm_pack(ntensors, tensors, numel, NORM_CHUNK, [&](const NormPack& pk, int used, uint32_t chunks) {
        const int blocks = chunks < VCR_OPT_NORM_BLOCKS ? (int)chunks : VCR_OPT_NORM_BLOCKS;
        if (*npartials + blocks > capacity) { vcr_set_error("vcr_grad_norm_accumulate: room for %d partial sums is too little", capacity); return 1; }
        const dim3 grid(blocks), block(256);
        double* out = partials + *npartials;
        if (type == VCR_F32) hipLaunchKernelGGL(norm_kernel<float>, grid, block, 0, (hipStream_t)stream, pk, used, NORM_CHUNK, out);
        else if (type == VCR_BF16) hipLaunchKernelGGL(norm_kernel<__hip_bfloat16>, grid, block, 0, (hipStream_t)stream, pk, used, NORM_CHUNK, out);
        else hipLaunchKernelGGL(norm_kernel<__half>, grid, block, 0, (hipStream_t)stream, pk, used, NORM_CHUNK, out);
        *npartials += blocks;
        return 0;
    });
    if (rc) return 1;
    VCR_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int vcr_grad_norm_finish(const double* partials, int npartials, double grad_scale, float* norm, void* stream) {
    if (!norm || npartials < 0 || (npartials > 0 && !partials)) { vcr_set_error("vcr_grad_norm_finish: partials or norm is NULL"); return 1; }
    hipLaunchKernelGGL(norm_final_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, partials, npartials, fabs(grad_scale), norm);
    VCR_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int vcr_clip_gradients(int ntensors, void* const* tensors, const int64_t* numel, int type, const float* norm, double max_norm,
                                  void* stream) {
    if (list_check("vcr_clip_gradients", ntensors, tensors, numel, type)) return 1;
    if (!norm) { vcr_set_error("vcr_clip_gradients: norm is NULL"); return 1; }
    const int rc = each_norm_pack(ntensors, (const void* const*)tensors, numel, NORM_CHUNK, [&](const NormPack& pk, int used, uint32_t chunks) {
        const dim3 grid(chunks < 4096 ? chunks : 4096), block(256);
        if (type == VCR_F32) hipLaunchKernelGGL(scale_kernel<float>, grid, block, 0, (hipStream_t)stream, pk, used, NORM_CHUNK, norm, max_norm);
        else if (type == VCR_BF16) hipLaunchKernelGGL(scale_kernel<__hip_bfloat16>, grid, block, 0, (hipStream_t)stream, pk, used, NORM_CHUNK, norm, max_norm);
        else hipLaunchKernelGGL(scale_kernel<__half>, grid, block, 0, (hipStream_t)stream, pk, used, NORM_CHUNK, norm, max_norm);
        return 0;
    });
    if (rc) return 1;
    VCR_HIP_CHECK(hipGetLastError());
    return 0;
}
