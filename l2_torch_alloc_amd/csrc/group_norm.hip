// Group norm with an activation, channels last, forward and backward, for gfx950.
//
//   mean, var over the pixels and channels of a (sample, group);  r = 1 / sqrt(var + eps)
//   h = (x - mean) r,   z = w h + b,   y = act(z)
//   dz = dout act'(z);  db = sum dz,  dw = sum dz h  (over samples and pixels)
//   dx = r (w dz - mean_g(w dz) - h mean_g(w dz h))  (means over the (sample, group))
//
// Bound by memory: the array must be read before the first value of its output is known, so it is read
// twice, the second time out of the caches where it fits them (a workgroup's own, or the Infinity Cache).
//
// A lane keeps one vector of channels and walks pixels, so all accesses of a wave are runs of whole
// vectors and its sums are per channel, in registers; whatever the number of channels in a group is,
// groups are only told apart when the sums are added up.  The sums of squares are of differences to
// the lane's first value of the channel, so that a mean far from zero costs no digits, and become
// doubles before lanes are added: every sum of doubles below is in a fixed order, so results do not
// depend on which workgroup came first.
#include <hip/hip_runtime.h>

#include "group_norm.h"

namespace sideaware {
namespace {

struct GnArgs {
    const void* x;
    const void* dout;
    void* out;
    const void* weight;
    const void* bias;
    float* stats;
    void* dweight;
    void* dbias;
    double* group_part;
    float* means;
    float* channel_part;
    long long batch, pixels, batch_blocks, channel_rows, main_blocks;
    double inv_count;               // 1 / (pixels * channels of a group)
    int channels, groups, group_channels, row_vectors;
    int slab_vectors, slabs, slab_groups, slice_vectors, rows, chunks;
    int weight_fp32, activation, finish;
    float eps;
};

// The values of a vector stay packed in whole words until they are used: as an array of 16-bit values each of
// them would take a register of its own.
template<int BYTES> struct Words { typedef unsigned int type __attribute__((ext_vector_type(BYTES / 4))); };
template<> struct Words<4> { typedef unsigned int type; };
template<> struct Words<2> { typedef unsigned short type; };

template<typename T, int VEC>
struct Vec {
    typename Words<(int)sizeof(T) * VEC>::type words;
    // (The empty statement keeps the compiler from unpacking a whole batch ahead of the branches that use it.)
    __device__ __forceinline__ void unpack(float (&to)[VEC]) const {
        T v[VEC];
        auto here = words;
        asm volatile("" : "+v"(here));
        __builtin_memcpy(v, &here, sizeof here);
        #pragma unroll
        for (int j = 0; j < VEC; j++) to[j] = (float)v[j];
    }
    __device__ __forceinline__ void pack(const float (&from)[VEC]) {
        T v[VEC];
        #pragma unroll
        for (int j = 0; j < VEC; j++) v[j] = (T)from[j];
        __builtin_memcpy(&words, v, sizeof words);
    }
};

// One parameter (weight or bias) of each of a lane's channels.  The vector may start anywhere a value may.
template<typename T, int VEC>
__device__ __forceinline__ void load_params(float (&to)[VEC], const void* p, int fp32, int c, float missing) {
    if (!p) {
        #pragma unroll
        for (int j = 0; j < VEC; j++) to[j] = missing;
    } else if (fp32) {
        const float* from = (const float*)p + c;
        #pragma unroll
        for (int j = 0; j < VEC; j++) to[j] = from[j];
    } else {
        const T* from = (const T*)p + c;
        #pragma unroll
        for (int j = 0; j < VEC; j++) to[j] = (float)from[j];
    }
}

template<typename T>
__device__ __forceinline__ void store_param(void* p, int fp32, int c, float value) {
    if (!p) return;
    if (fp32) ((float*)p)[c] = value;
    else ((T*)p)[c] = (T)value;
}

// 1 / (1 + e^-z): the hardware's exponential and reciprocal, one unit in the last place each (and the
// rounding of the exponent's argument, |z| 2^-24 of the result)
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// Where this workgroup works, and which vector of a slice and which row this lane has.
struct Place {
    long long n;                    // sample (its first, where a workgroup has several)
    int slab, chunk;
    int first_vector, end_vector;   // of the slab
    int first_group, groups;        // of the slab
    int tx, ty;
};

__device__ __forceinline__ Place place_of(const GnArgs& a, unsigned int block) {
    Place q;
    unsigned int rest = block;
    q.chunk = 0;
    if (a.chunks > 1) {
        rest = block / (unsigned int)a.chunks;
        q.chunk = (int)(block - rest * (unsigned int)a.chunks);
    }
    unsigned int n = rest;
    q.slab = 0;
    if (a.slabs > 1) {
        n = rest / (unsigned int)a.slabs;
        q.slab = (int)(rest - n * (unsigned int)a.slabs);
    }
    q.n = n;
    q.first_vector = q.slab * a.slab_vectors;
    q.end_vector = min(q.first_vector + a.slab_vectors, a.row_vectors);
    q.first_group = q.slab * a.slab_groups;
    q.groups = min(a.slab_groups, a.groups - q.first_group);
    q.ty = (int)threadIdx.x / a.slice_vectors;
    q.tx = (int)threadIdx.x - q.ty * a.slice_vectors;
    return q;
}

// The pixels of one lane in one slice: the `ty`-th of the chunk's runs of `rows` pixels.  A run's address is the
// same for all lanes, and a lane's offset from it has 32 bits (the plan sees to that).
template<typename T, int VEC>
struct Lane {
    typedef Vec<T, VEC> V;
    long long base, step;           // bytes from the array's start to the chunk's first run, and on to its next
    unsigned int off, off_last;     // bytes from a run's start to the lane's vector; in the last run, if some rows have
                                    // no pixel there, to the vector of one that has
    int runs, whole;                // of the chunk; those in which all rows have a pixel
    int count = 0;                  // the lane's pixels; 0: it has none
    int v;                          // vector of the row
    __device__ __forceinline__ Lane(const GnArgs& a, const Place& q, long long n, int v0) {
        const unsigned int stride = (unsigned int)a.chunks * (unsigned int)a.rows;
        const unsigned int first = (unsigned int)q.chunk * (unsigned int)a.rows;
        const unsigned int left = (unsigned int)a.pixels - first;
        whole = (int)(left / stride);
        unsigned int more = left - (unsigned int)whole * stride;         // pixels from the start of the last run
        runs = whole + (more > 0 ? 1 : 0);
        if (more >= (unsigned int)a.rows) { whole++; more = 0; }
        v = v0 + q.tx;
        base = (n * a.pixels + first) * a.row_vectors * (long long)sizeof(V);
        step = (long long)stride * a.row_vectors * (long long)sizeof(V);
        off = (unsigned int)(q.ty * a.row_vectors + v) * (unsigned int)sizeof(V);
        const bool in_last = whole == runs || (unsigned int)q.ty < more;
        off_last = in_last ? off : (unsigned int)v * (unsigned int)sizeof(V);
        if (q.ty < a.rows && v < min(v0 + a.slice_vectors, q.end_vector)) count = whole == runs || in_last ? runs : whole;
    }
    // B pixels from the i-th run on; behind the last one, and where the lane has none, some other, so that all
    // loads are made side by side with nothing to wait for in between
    template<bool NT = false, int B>
    __device__ __forceinline__ void load(V (&to)[B], const void* array, int i) const {
        #pragma unroll
        for (int u = 0; u < B; u++) to[u] = load<NT>(array, min(i + u, runs - 1));
    }
    template<bool NT = false>
    __device__ __forceinline__ V load(const void* array, int run) const {
        const auto* from = (const decltype(V::words)*)((const char*)array + base + run * step + (run < whole ? off : off_last));
        V to;
        to.words = NT ? __builtin_nontemporal_load(from) : *from;
        return to;
    }
    __device__ __forceinline__ void store(void* array, int i, const V& value) const {
        auto* to = (decltype(V::words)*)((char*)array + base + i * step + off);
#ifndef GN_ST
#define GN_ST 0
#endif
        if constexpr (GN_ST == 1 || (GN_ST >= 2 && sizeof(value.words) < 16)) __builtin_nontemporal_store(value.words, to);
        else if constexpr (GN_ST == 2) { auto w = value.words; asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" : : "v"(to), "v"(w) : "memory"); }
        else if constexpr (GN_ST == 3) { auto w = value.words; asm volatile("global_store_dwordx4 %0, %1, off sc1 nt\n\ts_nop 1" : : "v"(to), "v"(w) : "memory"); }
        else *to = value.words;
    }
};

// The slab's group (counted from its first) of each channel of a vector.
template<int VEC>
__device__ __forceinline__ void groups_of(int (&g)[VEC], const GnArgs& a, const Place& q, int v) {
    int at = v * VEC / a.group_channels, left = (at + 1) * a.group_channels - v * VEC;
    #pragma unroll
    for (int j = 0; j < VEC; j++) {
        g[j] = at - q.first_group;
        if (--left == 0) { at++; left = a.group_channels; }
    }
}

// Threads that share one of `groups` sums: a power of two, in one wave.
__device__ __forceinline__ int threads_per_group(int groups) {
    int per = 1;
    while (per < 64 && per * 2 * groups <= (int)blockDim.x) per *= 2;
    return per;
}

__device__ __forceinline__ double add_over(double t, int per) {
    for (int d = per / 2; d > 0; d /= 2) t += __shfl_xor(t, d, 64);
    return t;
}

// The sums of the chunks of a sample's slab, by the workgroup of any chunk: sums[group] = {S1, S2}.
__device__ __forceinline__ void gather_chunks(const GnArgs& a, const Place& q, double* lds, double (*sums)[2]) {
    const double* part = a.group_part + (q.n * a.slabs + q.slab) * a.chunks * a.slab_groups * 2;
    for (int base = 0; base < q.groups; base += (int)blockDim.x) {
        const int here = min(q.groups - base, (int)blockDim.x);
        const int per = (int)blockDim.x / here;                   // threads that share a group's chunks
        const int g = (int)threadIdx.x % here, part_of = (int)threadIdx.x / here;
        double s1 = 0, s2 = 0;
        if (part_of < per) {
            for (int k = part_of; k < a.chunks; k += per) {
                const double* at = part + ((long long)k * a.slab_groups + base + g) * 2;
                s1 += at[0];
                s2 += at[1];
            }
            lds[threadIdx.x * 2] = s1;
            lds[threadIdx.x * 2 + 1] = s2;
        }
        __syncthreads();
        if ((int)threadIdx.x < here) {
            s1 = s2 = 0;
            for (int i = 0; i < per; i++) {
                s1 += lds[(i * here + g) * 2];
                s2 += lds[(i * here + g) * 2 + 1];
            }
            sums[base + g][0] = s1;
            sums[base + g][1] = s2;
        }
        __syncthreads();
    }
}

__device__ __forceinline__ void clear_sums(const Place& q, double (*sums)[2]) {
    for (int g = (int)threadIdx.x; g < q.groups; g += (int)blockDim.x) sums[g][0] = sums[g][1] = 0;
    __syncthreads();
}

__device__ __forceinline__ void write_part(const GnArgs& a, const Place& q, double (*sums)[2]) {
    double* part = a.group_part + ((q.n * a.slabs + q.slab) * a.chunks + q.chunk) * a.slab_groups * 2;
    for (int g = (int)threadIdx.x; g < q.groups; g += (int)blockDim.x) {
        part[g * 2] = sums[g][0];
        part[g * 2 + 1] = sums[g][1];
    }
}

enum Mode { kSums, kApply, kBoth };

// All workgroups start together and would stay in step: every lane waiting for its batch of loads, then every lane
// computing and the memory idle.  So the load that follows on a pixel's heels is issued where that pixel's registers are
// free, and this keeps the compiler from collecting the loads again.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// ---- forward -----------------------------------------------------------------------------------

// Pixels whose loads a lane has in flight: as many as fit its registers without spilling.
constexpr int forward_batch(int mode) { return mode == kApply ? 4 : 6; }

// The sums of d = x - pivot and of d^2 over the lane's pixels, by channel.  The pivot is the lane's first
// value of the group a channel belongs to.
template<typename T, int VEC, int B>
__device__ __forceinline__ void forward_lane_sums(const GnArgs& a, const Lane<T, VEC>& lane, Vec<T, VEC> (&cur)[B], const int (&g)[VEC],
                                                  float (&pivot)[VEC], float (&s1)[VEC], float (&s2)[VEC]) {
    typedef Vec<T, VEC> V;
    float first[VEC];
    cur[0].unpack(first);
    #pragma unroll
    for (int j = 0; j < VEC; j++) {
        pivot[j] = j > 0 && g[j] == g[j > 0 ? j - 1 : 0] ? pivot[j > 0 ? j - 1 : 0] : first[j];
        s1[j] = s2[j] = 0;
    }
    auto add = [&](const V& in) {
        float x[VEC];
        in.unpack(x);
        #pragma unroll
        for (int j = 0; j < VEC; j++) {
            const float d = x[j] - pivot[j];
            s1[j] += d;
            s2[j] = fmaf(d, d, s2[j]);
        }
    };
    int i = 0;
    for (; i + 2 * B <= lane.whole; i += B) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            add(cur[u]);
            cur[u] = lane.load(a.x, i + B + u);
            in_order();
        }
    }
    #pragma unroll
    for (int u = 0; u < B; u++) {
        if (i + u < lane.count) add(cur[u]);
        if (i + B + u < lane.runs) {
            cur[u] = lane.load(a.x, i + B + u);
        }
        in_order();
    }
    i += B;
    if (i >= lane.runs) return;
    #pragma unroll
    for (int u = 0; u < B; u++) {
        if (i + u < lane.count) add(cur[u]);
    }
}

// Adds the lanes' sums up to the slab's groups.  A vector of channels touches one or two groups, or, where
// groups are narrower than it, up to VEC of them, which go through LDS two at a time: each lane leaves its
// two groups' sums there, and the threads of a group pick up those of the vectors it has a part in.
template<int VEC>
__device__ __forceinline__ void forward_group_sums(const GnArgs& a, const Place& q, int v0, int count, const int (&g)[VEC], const float (&pivot)[VEC],
                                                   const float (&s1)[VEC], const float (&s2)[VEC], double* lds, double (*sums)[2]) {
    const int passes = a.group_channels >= VEC ? 1 : (VEC / a.group_channels + 2) / 2;
    const int end = min(v0 + a.slice_vectors, q.end_vector);
    const int per = threads_per_group(q.groups);
    const int first = (int)threadIdx.x / per, part = (int)threadIdx.x % per, step = (int)blockDim.x / per;
    for (int pass = 0; pass < passes; pass++) {
        if (q.ty < a.rows) {
            double t[4] = {0, 0, 0, 0};
            if (count) {
                #pragma unroll
                for (int slot = 0; slot < 2; slot++) {
                    // the group's channels in fp32 still, all of one pivot; then x = pivot + d
                    float f1 = 0, f2 = 0, p = 0;
                    int values = 0;
                    #pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const bool in = g[j] - g[0] == 2 * pass + slot;
                        f1 += in ? s1[j] : 0.0f;
                        f2 += in ? s2[j] : 0.0f;
                        p = in ? pivot[j] : p;
                        values += in ? count : 0;
                    }
                    const double dp = p, m = values, df = f1;
                    t[2 * slot] = values ? df + m * dp : 0.0;
                    t[2 * slot + 1] = values ? f2 + dp * (2.0 * df + m * dp) : 0.0;
                }
            }
            double* to = lds + (q.ty * a.slice_vectors + q.tx) * 4;
            #pragma unroll
            for (int k = 0; k < 4; k++) to[k] = t[k];
        }
        __syncthreads();
        for (int base = 0; base < q.groups; base += step) {
            const int at = base + first;
            double t1 = 0, t2 = 0;
            if (at < q.groups) {
                const int c0 = (q.first_group + at) * a.group_channels;
                const int lo = max(c0 / VEC, v0), hi = min((c0 + a.group_channels - 1) / VEC + 1, end);
                for (int w = lo; w < hi; w++) {
                    const int slot = q.first_group + at - w * VEC / a.group_channels - 2 * pass;
                    if (slot == 0 || slot == 1) {
                        const double* from = lds + (w - v0) * 4 + slot * 2;
                        for (int row = part; row < a.rows; row += per) {
                            t1 += from[row * a.slice_vectors * 4];
                            t2 += from[row * a.slice_vectors * 4 + 1];
                        }
                    }
                }
            }
            t1 = add_over(t1, per);
            t2 = add_over(t2, per);
            if (at < q.groups && part == 0) {
                sums[at][0] += t1;
                sums[at][1] += t2;
            }
        }
        __syncthreads();
    }
}

// mean and 1/sqrt(var + eps) from the means of x and x^2
__device__ __forceinline__ void write_stats(float* to, double mean, double square, float eps) {
    double var = square - mean * mean;
    if (var < 0) var = 0;                                         // rounding; a NaN stays one
    to[0] = (float)mean;
    to[1] = (float)(1.0 / sqrt(var + (double)eps));
}

__device__ __forceinline__ void forward_stats(const GnArgs& a, const Place& q, long long n, double (*sums)[2], float (*stat)[2], bool write) {
    for (int g = (int)threadIdx.x; g < q.groups; g += (int)blockDim.x) {
        write_stats(stat[g], sums[g][0] * a.inv_count, sums[g][1] * a.inv_count, a.eps);
        if (write) {
            float* to = a.stats + (n * a.groups + q.first_group + g) * 2;
            to[0] = stat[g][0];
            to[1] = stat[g][1];
        }
    }
    __syncthreads();
}

// two floats of each of the slab's groups
__device__ __forceinline__ void load_stats(const float* from, const GnArgs& a, const Place& q, long long n, float (*stat)[2]) {
    const float* at = from + (n * a.groups + q.first_group) * 2;
    for (int g = (int)threadIdx.x; g < q.groups; g += (int)blockDim.x) {
        stat[g][0] = at[g * 2];
        stat[g][1] = at[g * 2 + 1];
    }
    __syncthreads();
}

template<typename T, int VEC, bool SILU, int B>
__device__ __forceinline__ void forward_apply(const GnArgs& a, const Lane<T, VEC>& lane, Vec<T, VEC> (&cur)[B], const float (&mean)[VEC],
                                              const float (&scale)[VEC], const float (&shift)[VEC]) {
    typedef Vec<T, VEC> V;
    auto one = [&](const V& in) {
        float x[VEC];
        in.unpack(x);
        #pragma unroll
        for (int j = 0; j < VEC; j++) {
            const float z = fmaf(x[j] - mean[j], scale[j], shift[j]);
            x[j] = SILU ? z * sigmoid(z) : z;
        }
        V o;
        o.pack(x);
        return o;
    };
    int i = 0;
    for (; i + 2 * B <= lane.whole; i += B) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            lane.store(a.out, i + u, one(cur[u]));
            cur[u] = lane.load(a.x, i + B + u);
            in_order();
        }
    }
    #pragma unroll
    for (int u = 0; u < B; u++) {
        if (i + u < lane.count) lane.store(a.out, i + u, one(cur[u]));
        if (i + B + u < lane.runs) {
            cur[u] = lane.load(a.x, i + B + u);
        }
        in_order();
    }
    i += B;
    if (i >= lane.runs) return;
    #pragma unroll
    for (int u = 0; u < B; u++) {
        if (i + u < lane.count) lane.store(a.out, i + u, one(cur[u]));
    }
}


template<typename T, int VEC, int MODE>
__global__ __launch_bounds__(kGroupNormMaxThreads, MODE == kBoth ? 2 : 4) void group_norm_forward(GnArgs a) {
    extern __shared__ double lds[];
    __shared__ double sums[kGroupNormMaxSlabGroups][2];
    __shared__ float stat[kGroupNormMaxSlabGroups][2];
    const Place q = place_of(a, blockIdx.x);
    for (long long n = q.n; n < a.batch; n += a.batch_blocks) {   // once, unless samples are shared out
        constexpr int B = forward_batch(MODE);
        Vec<T, VEC> pre[B];                                  // the first pixels of a slice
        // whether they are the first slice's when the values are applied
        const bool kept = MODE == kApply || q.end_vector - q.first_vector <= a.slice_vectors;
        float scale[VEC], shift[VEC];
        {
            // on their way before anything else is done
            const Lane<T, VEC> lane(a, q, n, q.first_vector);
            if (lane.count) {
                lane.load(pre, a.x, 0);
                if constexpr (MODE != kSums) {
                    load_params<T, VEC>(scale, a.weight, a.weight_fp32, lane.v * VEC, 1.0f);
                    load_params<T, VEC>(shift, a.bias, a.weight_fp32, lane.v * VEC, 0.0f);
                }
            }
        }
        if constexpr (MODE != kApply) {
            clear_sums(q, sums);
            for (int v0 = q.first_vector; v0 < q.end_vector; v0 += a.slice_vectors) {
                const Lane<T, VEC> lane(a, q, n, v0);
                float pivot[VEC], s1[VEC], s2[VEC];
                int g[VEC];
                if (lane.count) {
                    if (v0 != q.first_vector) lane.load(pre, a.x, 0);
                    groups_of<VEC>(g, a, q, lane.v);
                    if constexpr (MODE == kBoth) {
                        Vec<T, VEC> cur[B];                       // `pre` stays, to be applied
                        #pragma unroll
                        for (int u = 0; u < B; u++) cur[u] = pre[u];
                        forward_lane_sums<T, VEC, B>(a, lane, cur, g, pivot, s1, s2);
                    } else {
                        forward_lane_sums<T, VEC, B>(a, lane, pre, g, pivot, s1, s2);
                    }
                }
                forward_group_sums<VEC>(a, q, v0, lane.count, g, pivot, s1, s2, lds, sums);
            }
        }
        if constexpr (MODE == kSums) {
            write_part(a, q, sums);
            return;
        }
        if (MODE == kApply && a.finish) {
            load_stats(a.stats, a, q, n, stat);
        } else {
            if constexpr (MODE == kApply) gather_chunks(a, q, lds, sums);
            forward_stats(a, q, n, sums, stat, q.chunk == 0);
        }
        for (int v0 = q.first_vector; v0 < q.end_vector; v0 += a.slice_vectors) {
            const Lane<T, VEC> lane(a, q, n, v0);
            if (!lane.count) continue;
            if (!kept || v0 != q.first_vector) lane.load(pre, a.x, 0);
            if (v0 != q.first_vector) {
                load_params<T, VEC>(scale, a.weight, a.weight_fp32, lane.v * VEC, 1.0f);
                load_params<T, VEC>(shift, a.bias, a.weight_fp32, lane.v * VEC, 0.0f);
            }
            float mean[VEC];
            int g[VEC];
            groups_of<VEC>(g, a, q, lane.v);
            #pragma unroll
            for (int j = 0; j < VEC; j++) {
                mean[j] = stat[g[j]][0];
                scale[j] *= stat[g[j]][1];
            }
            if (a.activation == kGroupNormSilu) forward_apply<T, VEC, true, B>(a, lane, pre, mean, scale, shift);
            else forward_apply<T, VEC, false, B>(a, lane, pre, mean, scale, shift);
        }
        __syncthreads();
    }
}

// Adds up the chunks' sums of four groups of a sample and leaves what the last launch reads: forward the
// statistics, backward the two means.
template<bool BACKWARD>
__global__ __launch_bounds__(256) void group_norm_finish(GnArgs a) {
    __shared__ double lds[256 * 2];
    const unsigned int quads = (unsigned int)(a.slab_groups + 3) / 4;
    const unsigned int sample_slab = blockIdx.x / quads, quad = blockIdx.x - sample_slab * quads;
    const unsigned int n = sample_slab / (unsigned int)a.slabs, slab = sample_slab - n * (unsigned int)a.slabs;
    const int of = (int)threadIdx.x % 4, in_slab = (int)quad * 4 + of, g = (int)slab * a.slab_groups + in_slab;
    const bool on = in_slab < a.slab_groups && g < a.groups;
    double s1 = 0, s2 = 0;
    if (on) {
        const double* part = a.group_part + ((long long)sample_slab * a.chunks * a.slab_groups + in_slab) * 2;
        #pragma unroll 4
        for (int k = (int)threadIdx.x / 4; k < a.chunks; k += 64) {
            const double* at = part + (long long)k * a.slab_groups * 2;
            s1 += at[0];
            s2 += at[1];
        }
    }
    lds[threadIdx.x * 2] = s1;
    lds[threadIdx.x * 2 + 1] = s2;
    for (int half = 128; half >= 4; half /= 2) {
        __syncthreads();
        if ((int)threadIdx.x < half) {
            lds[threadIdx.x * 2] += lds[(threadIdx.x + half) * 2];
            lds[threadIdx.x * 2 + 1] += lds[(threadIdx.x + half) * 2 + 1];
        }
    }
    if (threadIdx.x < 4 && on) {
        s1 = lds[threadIdx.x * 2] * a.inv_count;
        s2 = lds[threadIdx.x * 2 + 1] * a.inv_count;
        float* to = (BACKWARD ? a.means : a.stats) + ((long long)n * a.groups + g) * 2;
        if constexpr (BACKWARD) {
            to[0] = (float)s1;
            to[1] = (float)s2;
        } else {
            write_stats(to, s1, s2, a.eps);
        }
    }
}

// ---- backward ----------------------------------------------------------------------------------

constexpr int backward_batch(int mode) { return mode == kBoth ? 3 : 2; }      // pixels of both arrays

// dz of a value from z
template<bool SILU>
__device__ __forceinline__ float grad_of_z(float dout, float z) {
    if constexpr (!SILU) return dout;
    const float s = sigmoid(z);
    return dout * (s * fmaf(z, 1.0f - s, 1.0f));
}

// What a lane needs of its channels to have z and dz of a value: z = (x - mean) scale + shift.
template<typename T, int VEC>
struct Channels {
    float mean[VEC], scale[VEC], shift[VEC];
    __device__ __forceinline__ void load(const GnArgs& a, const Place& q, long long n, int v, float (&rstd)[VEC]) {
        int g[VEC];
        load_params<T, VEC>(scale, a.weight, a.weight_fp32, v * VEC, 1.0f);
        load_params<T, VEC>(shift, a.bias, a.weight_fp32, v * VEC, 0.0f);
        groups_of<VEC>(g, a, q, v);
        const float2* stats = (const float2*)a.stats + n * a.groups + q.first_group;
        #pragma unroll
        for (int j = 0; j < VEC; j++) {
            const float2 s = stats[g[j]];
            mean[j] = s.x;
            rstd[j] = s.y;
            scale[j] *= s.y;
        }
    }
};

// The sums of dz and of dz h over the lane's pixels, by channel.
template<typename T, int VEC, bool SILU, int B>
__device__ __forceinline__ void backward_lane_sums(const GnArgs& a, const Place& q, long long n, const Lane<T, VEC>& lane,
                                                   Vec<T, VEC> (&x)[B], Vec<T, VEC> (&g)[B],
                                                   float (&s1)[VEC], float (&s2)[VEC]) {
    typedef Vec<T, VEC> V;
    Channels<T, VEC> ch;
    float rstd[VEC];
    ch.load(a, q, n, lane.v, rstd);
    #pragma unroll
    for (int j = 0; j < VEC; j++) s1[j] = s2[j] = 0;
    auto add = [&](const V& in, const V& grad) {
        float xs[VEC], gs[VEC];
        in.unpack(xs);
        grad.unpack(gs);
        #pragma unroll
        for (int j = 0; j < VEC; j++) {
            const float d = xs[j] - ch.mean[j];
            const float dz = grad_of_z<SILU>(gs[j], fmaf(d, ch.scale[j], ch.shift[j]));
            s1[j] += dz;
            s2[j] = fmaf(dz, d, s2[j]);
        }
    };
    int i = 0;
    for (; i + 2 * B <= lane.whole; i += B) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            add(x[u], g[u]);
            x[u] = lane.load(a.x, i + B + u);
            g[u] = lane.load(a.dout, i + B + u);
            in_order();
        }
    }
    #pragma unroll
    for (int u = 0; u < B; u++) {
        if (i + u < lane.count) add(x[u], g[u]);
        if (i + B + u < lane.runs) {
            x[u] = lane.load(a.x, i + B + u);
            g[u] = lane.load(a.dout, i + B + u);
        }
        in_order();
    }
    i += B;
    if (i < lane.runs) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            if (i + u < lane.count) add(x[u], g[u]);
        }
    }
    #pragma unroll
    for (int j = 0; j < VEC; j++) s2[j] *= rstd[j];
}

// Adds the lanes' sums up to channels (for the gradients of weight and bias, into `row` of the workspace) and
// those, weighted, to the slab's groups.
template<typename T, int VEC>
__device__ __forceinline__ void backward_group_sums(const GnArgs& a, const Place& q, int v0, bool on, const float (&s1)[VEC], const float (&s2)[VEC],
                                                    double* lds, double (*sums)[2], long long row, bool add_to_row) {
    const int slice_channels = a.slice_vectors * VEC;
    const int c0 = v0 * VEC, c1 = min(v0 + a.slice_vectors, q.end_vector) * VEC;
    float* lanes = (float*)lds;                                   // [row][channel of the slice]
    double* totals = lds + (a.rows * slice_channels + 1) / 2;     // [which][channel]
    float* to = a.channel_part + row * 2 * a.channels + c0;
    #pragma unroll
    for (int which = 0; which < 2; which++) {
        if (q.ty < a.rows) {
            float* at = lanes + q.ty * slice_channels + q.tx * VEC;
            #pragma unroll
            for (int j = 0; j < VEC; j++) at[j] = !on ? 0.0f : which ? s2[j] : s1[j];
        }
        __syncthreads();
        for (int c = (int)threadIdx.x; c < c1 - c0; c += (int)blockDim.x) {
            double t = 0;
            for (int r = 0; r < a.rows; r++) t += lanes[r * slice_channels + c];
            float* part = to + which * a.channels + c;
            *part = add_to_row ? *part + (float)t : (float)t;
            float w[1];
            load_params<T, 1>(w, a.weight, a.weight_fp32, c0 + c, 1.0f);
            totals[which * slice_channels + c] = t * w[0];
        }
        __syncthreads();
    }
    const int per = threads_per_group(q.groups);
    const int first = (int)threadIdx.x / per, part = (int)threadIdx.x % per, step = (int)blockDim.x / per;
    for (int base = 0; base < q.groups; base += step) {
        const int at = base + first;
        const int lo = max((q.first_group + at) * a.group_channels, c0), hi = min((q.first_group + at + 1) * a.group_channels, c1);
        double t1 = 0, t2 = 0;
        if (at < q.groups) {
            for (int c = lo + part; c < hi; c += per) {
                t1 += totals[c - c0];
                t2 += totals[slice_channels + c - c0];
            }
        }
        t1 = add_over(t1, per);
        t2 = add_over(t2, per);
        if (at < q.groups && part == 0) {
            sums[at][0] += t1;
            sums[at][1] += t2;
        }
    }
    __syncthreads();
}

// dx = rstd (w dz - c1 - h c2) as dz scale - (x - mean) e - d
template<typename T, int VEC, bool SILU, int B>
__device__ __forceinline__ void backward_apply(const GnArgs& a, const Place& q, long long n, const Lane<T, VEC>& lane,
                                               Vec<T, VEC> (&x)[B], Vec<T, VEC> (&g)[B], float (*stat)[2]) {
    typedef Vec<T, VEC> V;
    Channels<T, VEC> ch;
    float d[VEC], e[VEC];
    int gr[VEC];
    ch.load(a, q, n, lane.v, d);
    groups_of<VEC>(gr, a, q, lane.v);
    #pragma unroll
    for (int j = 0; j < VEC; j++) {
        e[j] = d[j] * d[j] * stat[gr[j]][1];
        d[j] *= stat[gr[j]][0];
    }
    auto one = [&](const V& in, const V& grad) {
        float xs[VEC], gs[VEC];
        in.unpack(xs);
        grad.unpack(gs);
        #pragma unroll
        for (int j = 0; j < VEC; j++) {
            const float m = xs[j] - ch.mean[j];
            const float dz = grad_of_z<SILU>(gs[j], fmaf(m, ch.scale[j], ch.shift[j]));
            xs[j] = fmaf(-m, e[j], fmaf(dz, ch.scale[j], -d[j]));
        }
        V o;
        o.pack(xs);
        return o;
    };
    int i = 0;
    for (; i + 2 * B <= lane.whole; i += B) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            lane.store(a.out, i + u, one(x[u], g[u]));
            x[u] = lane.load(a.x, i + B + u);
            g[u] = lane.load(a.dout, i + B + u);
            in_order();
        }
    }
    #pragma unroll
    for (int u = 0; u < B; u++) {
        if (i + u < lane.count) lane.store(a.out, i + u, one(x[u], g[u]));
        if (i + B + u < lane.runs) {
            x[u] = lane.load(a.x, i + B + u);
            g[u] = lane.load(a.dout, i + B + u);
        }
        in_order();
    }
    i += B;
    if (i >= lane.runs) return;
    #pragma unroll
    for (int u = 0; u < B; u++) {
        if (i + u < lane.count) lane.store(a.out, i + u, one(x[u], g[u]));
    }
}

// dw and db: the channels' sums added over the rows of the workspace, 64 channels to a workgroup.
template<typename T>
__device__ __forceinline__ void add_params(const GnArgs& a, long long block, double* lds) {
    constexpr int W = kGroupNormParamChannels;
    const int tx = (int)threadIdx.x % W, ty = (int)threadIdx.x / W, rows = (int)blockDim.x / W;
    const int c = (int)block * W + tx;
    double s1 = 0, s2 = 0;
    if (c < a.channels) {
        for (long long r = ty; r < a.channel_rows; r += rows) {
            s1 += a.channel_part[r * 2 * a.channels + c];
            s2 += a.channel_part[r * 2 * a.channels + a.channels + c];
        }
    }
    lds[threadIdx.x * 2] = s1;
    lds[threadIdx.x * 2 + 1] = s2;
    __syncthreads();
    if (ty == 0 && c < a.channels) {
        for (int i = 1; i < rows; i++) {
            s1 += lds[(i * W + tx) * 2];
            s2 += lds[(i * W + tx) * 2 + 1];
        }
        store_param<T>(a.dbias, a.weight_fp32, c, (float)s1);
        store_param<T>(a.dweight, a.weight_fp32, c, (float)s2);
    }
}

template<typename T, int VEC, int MODE>
__global__ __launch_bounds__(kGroupNormMaxThreads, MODE == kBoth ? 2 : 4) void group_norm_backward(GnArgs a) {
    extern __shared__ double lds[];
    __shared__ double sums[kGroupNormMaxSlabGroups][2];
    __shared__ float stat[kGroupNormMaxSlabGroups][2];
    if (MODE == kApply && blockIdx.x >= a.main_blocks) {
        add_params<T>(a, blockIdx.x - a.main_blocks, lds);
        return;
    }
    const Place q = place_of(a, blockIdx.x);
    const bool silu = a.activation == kGroupNormSilu;
    for (long long n = q.n; n < a.batch; n += a.batch_blocks) {
        constexpr int B = backward_batch(MODE);
        Vec<T, VEC> px[B], pg[B];
        const bool kept = MODE == kApply || q.end_vector - q.first_vector <= a.slice_vectors;
        {
            const Lane<T, VEC> lane(a, q, n, q.first_vector);
            if (lane.count) {
                lane.load(px, a.x, 0);
                lane.load(pg, a.dout, 0);
            }
        }
        if constexpr (MODE != kApply) {
            clear_sums(q, sums);
            for (int v0 = q.first_vector; v0 < q.end_vector; v0 += a.slice_vectors) {
                const Lane<T, VEC> lane(a, q, n, v0);
                float s1[VEC], s2[VEC];
                if (lane.count) {
                    if (v0 != q.first_vector) {
                        lane.load(px, a.x, 0);
                        lane.load(pg, a.dout, 0);
                    }
                    auto sum = [&](Vec<T, VEC> (&x)[B], Vec<T, VEC> (&g)[B]) {
                        if (silu) backward_lane_sums<T, VEC, true, B>(a, q, n, lane, x, g, s1, s2);
                        else backward_lane_sums<T, VEC, false, B>(a, q, n, lane, x, g, s1, s2);
                    };
                    if constexpr (MODE == kBoth) {
                        Vec<T, VEC> x[B], g[B];                   // `px` and `pg` stay, to be applied
                        #pragma unroll
                        for (int u = 0; u < B; u++) { x[u] = px[u]; g[u] = pg[u]; }
                        sum(x, g);
                    } else {
                        sum(px, pg);
                    }
                }
                backward_group_sums<T, VEC>(a, q, v0, lane.count != 0, s1, s2, lds, sums, q.n * a.chunks + q.chunk, n != q.n);
            }
        }
        if constexpr (MODE == kSums) {
            write_part(a, q, sums);
            return;
        }
        if (MODE == kApply && a.finish) {
            load_stats(a.means, a, q, n, stat);
        } else {
            if constexpr (MODE == kApply) gather_chunks(a, q, lds, sums);
            for (int g = (int)threadIdx.x; g < q.groups; g += (int)blockDim.x) {
                stat[g][0] = (float)(sums[g][0] * a.inv_count);
                stat[g][1] = (float)(sums[g][1] * a.inv_count);
            }
            __syncthreads();
        }
        for (int v0 = q.first_vector; v0 < q.end_vector; v0 += a.slice_vectors) {
            const Lane<T, VEC> lane(a, q, n, v0);
            if (!lane.count) continue;
            if (!kept || v0 != q.first_vector) {
                lane.load(px, a.x, 0);
                lane.load(pg, a.dout, 0);
            }
            if (silu) backward_apply<T, VEC, true, B>(a, q, n, lane, px, pg, stat);
            else backward_apply<T, VEC, false, B>(a, q, n, lane, px, pg, stat);
        }
        __syncthreads();
    }
}

template<typename T>
__global__ __launch_bounds__(256) void group_norm_params(GnArgs a) {
    __shared__ double lds[256 * 2];
    add_params<T>(a, blockIdx.x, lds);
}

// ---- launches ----------------------------------------------------------------------------------

GnArgs args_of(const GroupNormCall& c) {
    const GroupNormPlan& p = c.plan;
    GnArgs a = {};
    a.x = c.x; a.dout = c.dout; a.out = c.out; a.weight = c.weight; a.bias = c.bias; a.stats = c.stats;
    a.dweight = c.dweight; a.dbias = c.dbias;
    a.group_part = (double*)c.workspace;
    a.means = (float*)((char*)c.workspace + p.group_part_bytes);
    a.channel_part = (float*)((char*)c.workspace + p.group_part_bytes + p.means_bytes);
    a.batch = c.batch; a.pixels = c.pixels; a.batch_blocks = p.batch_blocks;
    a.channel_rows = p.channel_rows; a.main_blocks = p.blocks;
    a.inv_count = 1.0 / ((double)c.pixels * (double)p.group_channels);
    a.channels = c.channels; a.groups = c.groups; a.group_channels = p.group_channels; a.row_vectors = p.row_vectors;
    a.slab_vectors = p.slab_vectors; a.slabs = p.slabs; a.slab_groups = p.slab_groups; a.slice_vectors = p.slice_vectors;
    a.rows = p.rows; a.chunks = p.chunks;
    a.weight_fp32 = c.weight_fp32; a.activation = c.activation; a.finish = p.finish; a.eps = c.eps;
    return a;
}

template<typename T, int VEC>
hipError_t forward_of(const GroupNormCall& c, hipStream_t stream) {
    const GroupNormPlan& p = c.plan;
    const GnArgs a = args_of(c);
    const dim3 grid((unsigned)p.blocks), block((unsigned)p.threads);
    if (p.chunks == 1) {
        group_norm_forward<T, VEC, kBoth><<<grid, block, p.lds_bytes, stream>>>(a);
        return hipGetLastError();
    }
    group_norm_forward<T, VEC, kSums><<<grid, block, p.lds_bytes, stream>>>(a);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    if (p.finish) {
        group_norm_finish<false><<<dim3((unsigned)(c.batch * p.slabs * ((p.slab_groups + 3) / 4))), dim3(256), 0, stream>>>(a);
        err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    group_norm_forward<T, VEC, kApply><<<grid, block, p.lds_bytes, stream>>>(a);
    return hipGetLastError();
}

template<typename T, int VEC>
hipError_t backward_of(const GroupNormCall& c, hipStream_t stream) {
    const GroupNormPlan& p = c.plan;
    const GnArgs a = args_of(c);
    const dim3 grid((unsigned)p.blocks), block((unsigned)p.threads);
    if (p.chunks == 1) {
        group_norm_backward<T, VEC, kBoth><<<grid, block, p.lds_bytes, stream>>>(a);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess || (!c.dweight && !c.dbias)) return err;
        group_norm_params<T><<<dim3((unsigned)p.param_blocks), dim3(256), 0, stream>>>(a);
        return hipGetLastError();
    }
    group_norm_backward<T, VEC, kSums><<<grid, block, p.lds_bytes, stream>>>(a);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    if (p.finish) {
        group_norm_finish<true><<<dim3((unsigned)(c.batch * p.slabs * ((p.slab_groups + 3) / 4))), dim3(256), 0, stream>>>(a);
        err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    const dim3 both((unsigned)(p.blocks + (c.dweight || c.dbias ? p.param_blocks : 0)));
    group_norm_backward<T, VEC, kApply><<<both, block, p.lds_bytes, stream>>>(a);
    return hipGetLastError();
}

template<typename T, int VEC>
hipError_t launch_of(const GroupNormCall& c, bool backward, hipStream_t stream) {
    return backward ? backward_of<T, VEC>(c, stream) : forward_of<T, VEC>(c, stream);
}

template<typename T>
hipError_t launch_vec(const GroupNormCall& c, bool backward, hipStream_t stream) {
    switch (c.plan.vec) {
        case 1: return launch_of<T, 1>(c, backward, stream);
        case 2: return launch_of<T, 2>(c, backward, stream);
        case 4: return launch_of<T, 4>(c, backward, stream);
        case 8:
            if constexpr (sizeof(T) == 2) return launch_of<T, 8>(c, backward, stream);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_type(const GroupNormCall& c, bool backward, hipStream_t stream) {
    switch (c.type) {
        case kGroupNormFp32: return launch_vec<float>(c, backward, stream);
        case kGroupNormBf16: return launch_vec<__bf16>(c, backward, stream);
        case kGroupNormFp16: return launch_vec<_Float16>(c, backward, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace

int launch_group_norm_forward(const GroupNormCall& call, void* stream) { return (int)launch_type(call, false, (hipStream_t)stream); }
int launch_group_norm_backward(const GroupNormCall& call, void* stream) { return (int)launch_type(call, true, (hipStream_t)stream); }

}  // namespace sideaware
