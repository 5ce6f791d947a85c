// Host stand-ins for the device-side names that group_norm.hip uses, so that the whole file (kernels and the code that
// launches them) can be compiled for the CPU and run under sanitizers.  A workgroup's threads are threads of the host:
// barriers are real, lane moves go through an array of the wave.  Workgroups run one after another.
#pragma once
#include <pthread.h>

#include <cmath>
#include <cstddef>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <thread>
#include <vector>

#define __device__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static

struct dim3 {
    unsigned int x, y, z;
    dim3(unsigned int x = 1, unsigned int y = 1, unsigned int z = 1) : x(x), y(y), z(z) {}
};
struct alignas(8) float2 { float x, y; };
struct alignas(16) double2 { double x, y; };
typedef int hipError_t;
typedef void* hipStream_t;
constexpr hipError_t hipSuccess = 0, hipErrorInvalidValue = 1;
inline hipError_t hipGetLastError() { return hipSuccess; }

static thread_local dim3 threadIdx;
static dim3 blockIdx, blockDim, gridDim;

static char* cpu_lds;                                             // the launch's dynamic LDS: exactly as many bytes
static pthread_barrier_t cpu_block_barrier, cpu_wave_barrier[16];
static int64_t cpu_wave[16][64];
static long cpu_launches, cpu_chunked;

inline void __syncthreads() { pthread_barrier_wait(&cpu_block_barrier); }

// `v` of lane (lane ^ mask) of the wave
template<typename T>
T cpu_lane_xor(T v, unsigned int mask) {
    static_assert(sizeof(T) <= 8, "");
    const unsigned int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    std::memcpy(&cpu_wave[wave][lane], &v, sizeof v);
    pthread_barrier_wait(&cpu_wave_barrier[wave]);
    T got;
    std::memcpy(&got, &cpu_wave[wave][lane ^ mask], sizeof got);
    pthread_barrier_wait(&cpu_wave_barrier[wave]);
    return got;
}
inline int cpu_dpp(int v, int control) {
    // quad_perm [1,0,3,2] and [2,3,0,1], row_half_mirror, row_mirror
    return cpu_lane_xor(v, control == 0xB1 ? 1 : control == 0x4E ? 2 : control == 0x141 ? 7 : control == 0x140 ? 15 : (std::abort(), 0));
}
#define __builtin_amdgcn_update_dpp(old, v, control, rows, banks, bound) cpu_dpp(v, control)
inline double __shfl_xor(double v, int mask, int) { return cpu_lane_xor(v, (unsigned int)mask); }
inline int __double2hiint(double d) { int64_t b; std::memcpy(&b, &d, 8); return (int)(b >> 32); }
inline int __double2loint(double d) { int64_t b; std::memcpy(&b, &d, 8); return (int)(b & 0xffffffff); }
inline double __hiloint2double(int hi, int lo) {
    const uint64_t b = ((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo;
    double d;
    std::memcpy(&d, &b, 8);
    return d;
}
inline float __builtin_amdgcn_rcpf(float v) { return 1.0f / v; }
inline float __expf(float v) { return std::exp(v); }
#define __builtin_amdgcn_sched_barrier(x) ((void)0)
template<typename A, typename B> auto min(A a, B b) { return a < b ? a : b; }
template<typename A, typename B> auto max(A a, B b) { return a > b ? a : b; }

template<typename F, typename Args>
void cpu_launch(F kernel, const Args& args, dim3 grid, dim3 block, size_t lds_bytes, hipStream_t) {
    cpu_launches++;
    if (grid.x > 1) cpu_chunked++;
    gridDim = grid;
    blockDim = block;
    void* lds = nullptr;
    if (posix_memalign(&lds, 16, lds_bytes ? lds_bytes : 16) != 0 || block.x % 64 || block.x > 1024) std::abort();
    cpu_lds = (char*)lds;
    pthread_barrier_init(&cpu_block_barrier, nullptr, block.x);
    for (unsigned int w = 0; w < block.x / 64; w++) pthread_barrier_init(&cpu_wave_barrier[w], nullptr, 64);
    std::vector<std::thread> threads;
    for (unsigned int t = 0; t < block.x; t++) {
        threads.emplace_back([&, t] {
            threadIdx = dim3(t, 0, 0);
            for (unsigned int z = 0; z < grid.z; z++)
                for (unsigned int y = 0; y < grid.y; y++)
                    for (unsigned int x = 0; x < grid.x; x++) {
                        if (t == 0) {
                            blockIdx = dim3(x, y, z);
                            if (lds_bytes) std::memset(cpu_lds, 0xff, lds_bytes);        // NaN: nobody has written it
                        }
                        __syncthreads();
                        kernel(args);
                        __syncthreads();
                    }
        });
    }
    for (auto& t : threads) t.join();
    pthread_barrier_destroy(&cpu_block_barrier);
    for (unsigned int w = 0; w < block.x / 64; w++) pthread_barrier_destroy(&cpu_wave_barrier[w]);
    std::free(lds);
}
