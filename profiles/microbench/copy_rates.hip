// Rates under the floors of the optimizer operators: a non-temporal copy, and the bare access pattern of the fp32 AdamW update (four
// arrays read, three of them written).  1 GiB an array, 16 bytes a lane, one access a thread; 20 launches between two events.
// hipcc --offload-arch=gfx950 -O3 -Xclang -target-feature -Xclang -packed-fp32-ops -o copy_rates copy_rates.hip && ./copy_rates
#include <hip/hip_runtime.h>
#include <stdio.h>

typedef float f4 __attribute__((ext_vector_type(4)));
#define CHECK(x) do { hipError_t e_ = (x); if (e_ != hipSuccess) { fprintf(stderr, "%s: %s\n", #x, hipGetErrorString(e_)); return 1; } } while (0)

__global__ void __launch_bounds__(256) copy_kernel(const f4* a, f4* b) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    __builtin_nontemporal_store(__builtin_nontemporal_load(a + i), b + i);
}
__global__ void __launch_bounds__(256) update_kernel(f4* a, f4* b, f4* c, const f4* g) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const f4 x = __builtin_nontemporal_load(a + i), y = __builtin_nontemporal_load(b + i), z = __builtin_nontemporal_load(c + i);
    const f4 w = __builtin_nontemporal_load(g + i);
    __builtin_nontemporal_store(x + w, a + i);
    __builtin_nontemporal_store(y + w, b + i);
    __builtin_nontemporal_store(z + w, c + i);
}

int main() {
    const size_t n = 1ull << 26;          // (a multiple of the 256 threads of a workgroup: no tail)
    f4* p[4];
    for (auto& q : p) { CHECK(hipMalloc(&q, n * sizeof(f4))); CHECK(hipMemset(q, 0, n * sizeof(f4))); }
    hipEvent_t s, e;
    CHECK(hipEventCreate(&s));
    CHECK(hipEventCreate(&e));
    float ms;
    for (int r = 0; r < 4; ++r) {
        CHECK(hipEventRecord(s));
        for (int k = 0; k < 20; ++k) hipLaunchKernelGGL(copy_kernel, dim3(n / 256), dim3(256), 0, 0, p[0], p[1]);
        CHECK(hipEventRecord(e));
        CHECK(hipEventSynchronize(e));
        CHECK(hipEventElapsedTime(&ms, s, e));
        printf("copy                        %.0f GB/s\n", 20.0 * n * 32 / ms / 1e6);
        CHECK(hipEventRecord(s));
        for (int k = 0; k < 20; ++k) hipLaunchKernelGGL(update_kernel, dim3(n / 256), dim3(256), 0, 0, p[0], p[1], p[2], p[3]);
        CHECK(hipEventRecord(e));
        CHECK(hipEventSynchronize(e));
        CHECK(hipEventElapsedTime(&ms, s, e));
        printf("four read, three written    %.0f GB/s\n", 20.0 * n * 112 / ms / 1e6);
    }
    return 0;
}
