// Group norm with an activation, channels last, forward and backward, for gfx950.
//
//   mean, var over the pixels and channels of a (sample, group);  r = 1 / sqrt(var + eps)
//   h = (x - mean) r,   z = w h + b,   y = act(z)
//   dz = dout act'(z);  db = sum dz,  dw = sum dz h  (over samples and pixels)
//   dx = r (w dz - mean_g(w dz) - h mean_g(w dz h))  (means over the (sample, group))
//
// Bound by memory: the array must be read before the first value of its output is known, so it is read twice, the
// second time out of the caches where it fits them (a workgroup's own, or the Infinity Cache).  Forward, bf16 with SiLU
// and fp32 parameters: 512x512 pixels of 256 channels (134 MB) 73 us, 3.7 TB/s of what has to be read and written, of
// which 25 us for the sums (memory), 5 for adding the chunks' sums and 43 for the values (6.2 TB/s of what they read and
// write); 8 samples of 64x64 pixels of 320 channels (21 MB) 17 us, 8 and 9 for the two launches, of which about 3 us each
// go into adding sums up across lanes and workgroups.  Backward with SiLU is bound by the vector ALU too: 21 issue
// slots a value for the sums, of which an exponential and a reciprocal take eight; 16 samples of 32x32 pixels of 640
// channels (21 MB) 26 us, 2.4 TB/s.
//
// A lane keeps one vector of channels and walks pixels, so all accesses of a wave are runs of whole
// vectors and its sums are per channel, in registers; whatever the number of channels in a group is,
// groups are only told apart when the sums are added up.  The sums of squares are of differences to
// the lane's first value of the channel's group, so that a mean far from zero costs no digits, and become
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
    long long batch, pixels, channel_rows;
    double inv_count;               // 1 / (pixels * channels of a group)
    float inv_group_channels;
    float eps;
    unsigned int inv_slice, inv_gather;      // 2^20 / slice_vectors and / gather_groups, rounded up: for thread numbers below 512
    int channels, groups, group_channels, row_vectors;
    int slab_vectors, slab_groups, slice_vectors, rows, chunks;
    int runs, more_runs;            // runs of pixels of every chunk; the first `more_runs` chunks have one more
    int last_chunk, last_pixels;    // the chunk whose last run is not whole, and its pixels; -1 and 0: all are whole
    int gather_groups, gather_threads;       // groups whose chunks' sums are added at once, and threads to each
    int per_group_log2;             // threads to a group where lanes' sums are added
    int param_x, param_blocks;      // workgroups of a row of the grid that add up dw and db, and how many do in all
    int weight_fp32, activation, finish;
    int straddle;                   // a vector may hold channels of two groups
    int passes;                     // over the lanes' sums, two groups of every vector at a time
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

// Stores are written through the private L2 (`sc1`), which spares the end of the launch the write-backs: 22.2 us against
// 24.1 for 8 images of 64x64 pixels of 320 bf16 channels.  Where the arrays together exceed the Infinity Cache the
// output is not kept there either (`nt`): what the next call reads then does not wait for this one's output to be
// written back (512x512 pixels of 256 channels: 78 us against 88).  Narrow vectors are left to the L2, which may merge them.
// The two wait states: hardware reads the data registers of a store wider than 8 bytes for two more issue cycles, and the
// compiler does not look inside the statement.
// So are the pieces of memory lines that a workgroup with some of a row's channels writes, where its neighbours on the
// same XCD write the rest (64 samples of 1024 pixels of 512 channels: 31.6 us, 33.8 written through).
enum Store { kThrough, kStream, kMerge };
template<int STORE, typename W>
__device__ __forceinline__ void store_words(void* to, const W& words) {
    if constexpr (sizeof(W) == 16 && STORE != kMerge) {
        if constexpr (STORE == kStream) asm volatile("global_store_dwordx4 %0, %1, off sc1 nt\n\ts_nop 1" : : "v"(to), "v"(words) : "memory");
        else asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" : : "v"(to), "v"(words) : "memory");
    } else if constexpr (STORE == kStream) {
        __builtin_nontemporal_store(words, (W*)to);
    } else {
        *(W*)to = words;
    }
}

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

// The grid is (chunks, slabs, samples).  Workgroups are dealt to the XCDs in turn; those of one launch (NEAR), whose slabs are
// pieces of rows, are numbered so that each XCD has consecutive ones: a memory line is then fetched into one L2
// alone (16 samples of 256 pixels of 640 channels: 8.7 us dealt in turn, 7.5 so).
template<bool NEAR>
__device__ __forceinline__ Place place_of(const GnArgs& a, int chunk) {
    Place q;
    q.chunk = chunk;
    q.slab = (int)blockIdx.y;
    q.n = blockIdx.z;
    if constexpr (NEAR) {
        unsigned int at = blockIdx.z * gridDim.y + blockIdx.y;
        const unsigned int each = gridDim.y * gridDim.z / 8;
        if (at < each * 8) at = at % 8 * each + at / 8;
        q.n = at / gridDim.y;
        q.slab = (int)(at % gridDim.y);
    }
    q.first_vector = q.slab * a.slab_vectors;
    q.end_vector = min(q.first_vector + a.slab_vectors, a.row_vectors);
    q.first_group = q.slab * a.slab_groups;
    q.groups = min(a.slab_groups, a.groups - q.first_group);
    q.ty = (int)((threadIdx.x * a.inv_slice) >> 20);
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
        runs = a.runs + (q.chunk < a.more_runs ? 1 : 0);
        whole = q.chunk == a.last_chunk ? runs - 1 : runs;
        v = v0 + q.tx;
        const long long vector = sizeof(V);
        base = (n * a.pixels + (long long)q.chunk * a.rows) * a.row_vectors * vector;
        step = (long long)a.chunks * a.rows * a.row_vectors * vector;
        off = (unsigned int)(q.ty * a.row_vectors + v) * (unsigned int)sizeof(V);
        const bool in_last = whole == runs || q.ty < a.last_pixels;
        off_last = in_last ? off : (unsigned int)v * (unsigned int)sizeof(V);
        if (q.ty < a.rows && v < min(v0 + a.slice_vectors, q.end_vector)) count = in_last ? runs : whole;
    }
    // B pixels from the i-th run on; behind the last one, and where the lane has none, some other, so that all
    // loads are made side by side with nothing to wait for in between
    template<int B>
    __device__ __forceinline__ void load(V (&to)[B], const void* array, int i) const {
        #pragma unroll
        for (int u = 0; u < B; u++) to[u] = load(array, min(i + u, runs - 1));
    }
    __device__ __forceinline__ V load(const void* array, int run) const {
        return *(const V*)((const char*)array + base + run * step + (run < whole ? off : off_last));
    }
    template<int STORE>
    __device__ __forceinline__ void store(void* array, int i, const V& value) const {
        store_words<STORE>((char*)array + base + i * step + off, value.words);
    }
};

// The slab's group of its channel c: by a reciprocal, which is off by one at most.
__device__ __forceinline__ int group_of(const GnArgs& a, int c) {
    int g = (int)((float)c * a.inv_group_channels);
    if (g * a.group_channels > c) g--;
    if ((g + 1) * a.group_channels <= c) g++;
    return g;
}

// The slab's group of each channel of a vector.
template<int VEC>
__device__ __forceinline__ void groups_of(int (&g)[VEC], const GnArgs& a, const Place& q, int v) {
    const int c = (v - q.first_vector) * VEC;
    int at = group_of(a, c), left = (at + 1) * a.group_channels - c;
    #pragma unroll
    for (int j = 0; j < VEC; j++) {
        g[j] = at;
        if (--left == 0) { at++; left = a.group_channels; }
    }
}

template<int CTRL>
__device__ __forceinline__ double moved(double t) {
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(t), CTRL, 0xf, 0xf, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(t), CTRL, 0xf, 0xf, false));
}

// The sum over 2^per_log2 neighbouring threads of a wave, to all of them: moves inside a row of 16 lanes run in the
// vector ALU.
__device__ __forceinline__ double add_over(double t, int per_log2) {
    if (per_log2 > 0) t += moved<0xB1>(t);                        // quad_perm [1,0,3,2]
    if (per_log2 > 1) t += moved<0x4E>(t);                        // quad_perm [2,3,0,1]
    if (per_log2 > 2) t += moved<0x141>(t);                       // row_half_mirror: the other quad, all of it alike
    if (per_log2 > 3) t += moved<0x140>(t);                       // row_mirror: the other half of the row
    if (per_log2 > 4) t += __shfl_xor(t, 16, 64);
    if (per_log2 > 5) t += __shfl_xor(t, 32, 64);
    return t;
}

// The sums of the chunks of a sample's slab, by the workgroup of any chunk: sums[group] = {S1, S2}.
__device__ __forceinline__ void gather_chunks(const GnArgs& a, const Place& q, long long n, double* lds, double (*sums)[2]) {
    const double2* part = (const double2*)a.group_part + (n * gridDim.y + q.slab) * a.chunks * a.slab_groups;
    double2* lanes = (double2*)lds;
    const int share = (int)((threadIdx.x * a.inv_gather) >> 20), in = (int)threadIdx.x - share * a.gather_groups;
    for (int base = 0; base < q.groups; base += a.gather_groups) {
        const int g = base + in;
        if (share < a.gather_threads) {
            double2 t = {0, 0};
            if (g < q.groups) {
                // eight at a time, so that they are waited for once
                for (int k = share; k < a.chunks; k += 8 * a.gather_threads) {
                    double2 in4[8];
                    #pragma unroll
                    for (int u = 0; u < 8; u++) in4[u] = part[(long long)min(k + u * a.gather_threads, a.chunks - 1) * a.slab_groups + g];
                    #pragma unroll
                    for (int u = 0; u < 8; u++) {
                        const bool on = k + u * a.gather_threads < a.chunks;
                        t.x += on ? in4[u].x : 0.0;
                        t.y += on ? in4[u].y : 0.0;
                    }
                }
            }
            lanes[threadIdx.x] = t;
        }
        __syncthreads();
        if ((int)threadIdx.x < a.gather_groups && g < q.groups) {
            double2 t = {0, 0};
            #pragma unroll 4
            for (int i = 0; i < a.gather_threads; i++) {
                const double2 more = lanes[i * a.gather_groups + in];
                t.x += more.x;
                t.y += more.y;
            }
            sums[g][0] = t.x;
            sums[g][1] = t.y;
        }
        __syncthreads();
    }
}

__device__ __forceinline__ void clear_sums(const Place& q, double (*sums)[2]) {
    for (int g = (int)threadIdx.x; g < q.groups; g += (int)blockDim.x) sums[g][0] = sums[g][1] = 0;
    __syncthreads();
}

__device__ __forceinline__ void write_part(const GnArgs& a, const Place& q, long long n, double (*sums)[2]) {
    double* part = a.group_part + ((n * gridDim.y + q.slab) * a.chunks + q.chunk) * a.slab_groups * 2;
    for (int g = (int)threadIdx.x; g < q.groups; g += (int)blockDim.x) {
        part[g * 2] = sums[g][0];
        part[g * 2 + 1] = sums[g][1];
    }
}

// kApplyStream: as kApply, where the arrays exceed the Infinity Cache.  kBothMerge: as kBoth, where workgroups share
// memory lines.
enum Mode { kSums, kApply, kApplyStream, kBoth, kBothMerge };
constexpr bool does_both(int mode) { return mode == kBoth || mode == kBothMerge; }
constexpr int store_of(int mode) { return mode == kApplyStream ? kStream : mode == kBothMerge ? kMerge : kThrough; }
constexpr bool applies_only(int mode) { return mode == kApply || mode == kApplyStream; }

// All workgroups start together and would stay in step: every lane waiting for its batch of loads, then every lane
// computing and the memory idle.  So the load that follows on a pixel's heels is issued where that pixel's registers are
// free, and this keeps the compiler from collecting the loads again (64 samples of 256 pixels of 512 channels: 17 us, 19
// in batches).  The loops are not unrolled further and their last steps are loops of their own: with fewer instructions to
// fetch, a call of few values is faster (16 samples of one pixel: 6.7 us with batches of 2, 7.8 with batches of 6).
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// ---- forward -----------------------------------------------------------------------------------

// Pixels whose loads a lane has in flight: as many as fit its registers without spilling.
constexpr int forward_batch(int mode) { return applies_only(mode) ? 3 : 4; }

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
    #pragma unroll 1
    for (; i + 2 * B <= lane.whole; i += B) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            add(cur[u]);
            cur[u] = lane.load(a.x, i + B + u);
            in_order();
        }
    }
    #pragma unroll 1
    for (; i < lane.runs; i += B) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            if (i + u < lane.count) add(cur[u]);
            if (i + B + u < lane.runs) {
                cur[u] = lane.load(a.x, i + B + u);
            }
        }
    }
}

// Adds the lanes' sums up to the slab's groups.  A vector of channels touches one or two groups, or, where groups are
// narrower than it, up to VEC of them (gn_groups_of_vector), which go through LDS two at a time: each lane leaves its two
// groups' sums there, and the threads of a group pick up those of the vectors it has a part in.  (2 samples of 64 bf16 pixels of
// 32 groups: two passes, 5 channels each, 7.1 us; one pass, 6 channels each, 5.1.)
template<int VEC>
__device__ __forceinline__ void forward_group_sums(const GnArgs& a, const Place& q, int v0, int count, const int (&g)[VEC], const float (&pivot)[VEC],
                                                   const float (&s1)[VEC], const float (&s2)[VEC], double* lds, double (*sums)[2]) {
    const int end = min(v0 + a.slice_vectors, q.end_vector) - q.first_vector, start = v0 - q.first_vector;   // vectors of the slab
    const int per = 1 << a.per_group_log2;
    const int first = (int)threadIdx.x >> a.per_group_log2, part = (int)threadIdx.x & (per - 1), step = (int)blockDim.x >> a.per_group_log2;
    for (int pass = 0; pass < a.passes; pass++) {
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
                const int c0 = at * a.group_channels;
                const int lo = max(c0 / VEC, start), hi = min((c0 + a.group_channels - 1) / VEC + 1, end);
                for (int w = lo; w < hi; w++) {
                    // which of its vector's groups this one is (with one pass a vector has two at most)
                    int slot = w * VEC < c0 ? 1 : 0;
                    if (a.passes > 1) slot = at - group_of(a, w * VEC) - 2 * pass;
                    if (slot == 0 || slot == 1) {
                        const double* from = lds + (w - start) * 4 + slot * 2;
                        #pragma unroll 2
                        for (int row = part; row < a.rows; row += per) {
                            t1 += from[row * a.slice_vectors * 4];
                            t2 += from[row * a.slice_vectors * 4 + 1];
                        }
                    }
                }
            }
            t1 = add_over(t1, a.per_group_log2);
            t2 = add_over(t2, a.per_group_log2);
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
    to[1] = 1.0f / sqrtf((float)(var + (double)eps));             // three roundings of half a step
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

// What becomes of a group's two sums as soon as one thread has them, where nothing else adds to them: a chunk's go to
// the workspace, a sample's become its statistics.
template<int MODE>
__device__ __forceinline__ void forward_emit(const GnArgs& a, const Place& q, long long n, int at, double t1, double t2, float (*stat)[2]) {
    if constexpr (MODE == kSums) {
        double2* part = (double2*)a.group_part + ((n * gridDim.y + q.slab) * a.chunks + q.chunk) * a.slab_groups;
        part[at] = {t1, t2};
    } else {
        float s[2];
        write_stats(s, t1 * a.inv_count, t2 * a.inv_count, a.eps);
        *(float2*)stat[at] = {s[0], s[1]};
        ((float2*)a.stats)[n * a.groups + q.first_group + at] = {s[0], s[1]};
    }
}

// forward_group_sums() for one slice and groups no narrower than a vector, which then touches one group, or two where
// groups are no multiple of it (`straddle`): nothing is accumulated in between, so each group's threads pass its sums on.
template<int VEC, int MODE>
__device__ __forceinline__ void forward_group_sums_at_once(const GnArgs& a, const Place& q, long long n, int count, const int (&g)[VEC],
                                                           const float (&pivot)[VEC], const float (&s1)[VEC], const float (&s2)[VEC], double* lds,
                                                           float (*stat)[2]) {
    const int slots = a.straddle ? 2 : 1;
    double2* lanes = (double2*)lds;                               // [row][vector][slot]
    if (q.ty < a.rows) {
        double2* to = lanes + (q.ty * a.slice_vectors + q.tx) * slots;
        auto leave = [&](int slot, float f1, float f2, float p, int values) {
            const double dp = p, m = values, df = f1;
            double2 t = {df + m * dp, f2 + dp * (2.0 * df + m * dp)};
            if (values == 0) t = {0, 0};
            to[slot] = t;
        };
        float f1 = 0, f2 = 0;
        if (!a.straddle) {
            #pragma unroll
            for (int j = 0; j < VEC; j++) { f1 += s1[j]; f2 += s2[j]; }
            leave(0, f1, f2, pivot[0], VEC * count);
        } else {
            float h1 = 0, h2 = 0;
            int in = 0;
            #pragma unroll
            for (int j = 0; j < VEC; j++) {
                const bool first = g[j] == g[0];
                f1 += first ? s1[j] : 0.0f;
                f2 += first ? s2[j] : 0.0f;
                h1 += first ? 0.0f : s1[j];
                h2 += first ? 0.0f : s2[j];
                in += first ? count : 0;
            }
            leave(0, f1, f2, pivot[0], in);
            leave(1, h1, h2, pivot[VEC - 1], VEC * count - in);
        }
    }
    __syncthreads();
    const int per = 1 << a.per_group_log2;
    const int first = (int)threadIdx.x >> a.per_group_log2, part = (int)threadIdx.x & (per - 1), step = (int)blockDim.x >> a.per_group_log2;
    const int end = q.end_vector - q.first_vector;
    for (int base = 0; base < q.groups; base += step) {
        const int at = base + first;
        double t1 = 0, t2 = 0;
        if (at < q.groups) {
            const int c0 = at * a.group_channels, lo = c0 / VEC, vectors = min((c0 + a.group_channels - 1) / VEC + 1, end) - lo;
            const float inv = __builtin_amdgcn_rcpf((float)vectors);
            #pragma unroll 2
            for (int e = part; e < vectors * a.rows; e += per) {
                int row = (int)((float)e * inv);                  // e / vectors, off by one at most
                if (row * vectors > e) row--;
                if ((row + 1) * vectors <= e) row++;
                const int w = lo + e - row * vectors;
                const double2 t = lanes[(row * a.slice_vectors + w) * slots + (w * VEC < c0 ? 1 : 0)];
                t1 += t.x;
                t2 += t.y;
            }
        }
        t1 = add_over(t1, a.per_group_log2);
        t2 = add_over(t2, a.per_group_log2);
        if (at < q.groups && part == 0) forward_emit<MODE>(a, q, n, at, t1, t2, stat);
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

template<typename T, int VEC, bool SILU, int STORE, int B>
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
    #pragma unroll 1
    for (; i + 2 * B <= lane.whole; i += B) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            lane.template store<STORE>(a.out, i + u, one(cur[u]));
            cur[u] = lane.load(a.x, i + B + u);
            in_order();
        }
    }
    #pragma unroll 1
    for (; i < lane.runs; i += B) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            if (i + u < lane.count) lane.template store<STORE>(a.out, i + u, one(cur[u]));
            if (i + B + u < lane.runs) {
                cur[u] = lane.load(a.x, i + B + u);
            }
        }
    }
}


// kOne: a workgroup has one sample and its slab is one slice, as nearly always; the loops over them then go, and with
// them the registers that what they repeat would hold.  kOneWide: groups are no narrower than a vector, too.
enum Kind { kLoops, kOne, kOneWide };

template<typename T, int VEC, int MODE, int KIND>
__global__ __launch_bounds__(kGroupNormMaxThreads, 4) void group_norm_forward(GnArgs a) {
    constexpr bool ONE = KIND != kLoops, AT_ONCE = KIND == kOneWide;
    extern __shared__ __attribute__((aligned(16))) double lds[];
    __shared__ double sums[kGroupNormMaxSlabGroups][2];
    __shared__ __attribute__((aligned(8))) float stat[kGroupNormMaxSlabGroups][2];
    const Place q = place_of<does_both(MODE)>(a, (int)blockIdx.x);
    long long n = q.n;
    do {
        constexpr int B = forward_batch(MODE);
        Vec<T, VEC> pre[B];                                       // the first pixels of a slice
        // whether they are the first slice's when the values are applied
        const bool kept = ONE || applies_only(MODE) || q.end_vector - q.first_vector <= a.slice_vectors;
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
        if constexpr (!applies_only(MODE)) {
            if constexpr (!AT_ONCE) clear_sums(q, sums);
            int v0 = q.first_vector;
            do {
                const Lane<T, VEC> lane(a, q, n, v0);
                float pivot[VEC], s1[VEC], s2[VEC];
                int g[VEC];
                if (lane.count) {
                    if (!ONE && v0 != q.first_vector) lane.load(pre, a.x, 0);
                    groups_of<VEC>(g, a, q, lane.v);
                    if constexpr (does_both(MODE)) {
                        Vec<T, VEC> cur[B];                       // `pre` stays, to be applied
                        #pragma unroll
                        for (int u = 0; u < B; u++) cur[u] = pre[u];
                        forward_lane_sums<T, VEC, B>(a, lane, cur, g, pivot, s1, s2);
                    } else {
                        forward_lane_sums<T, VEC, B>(a, lane, pre, g, pivot, s1, s2);
                    }
                }
                if constexpr (AT_ONCE) forward_group_sums_at_once<VEC, MODE>(a, q, n, lane.count, g, pivot, s1, s2, lds, stat);
                else forward_group_sums<VEC>(a, q, v0, lane.count, g, pivot, s1, s2, lds, sums);
                v0 += a.slice_vectors;
            } while (!ONE && v0 < q.end_vector);
        }
        if constexpr (MODE == kSums) {
            if constexpr (!AT_ONCE) write_part(a, q, n, sums);
        } else {
            if (applies_only(MODE) && a.finish) {
                load_stats(a.stats, a, q, n, stat);
            } else if constexpr (applies_only(MODE) || !AT_ONCE) {
                if constexpr (applies_only(MODE)) gather_chunks(a, q, n, lds, sums);
                forward_stats(a, q, n, sums, stat, q.chunk == 0);
            }
            int v0 = q.first_vector;
            do {
                const Lane<T, VEC> lane(a, q, n, v0);
                if (lane.count) {
                    if (!kept || (!ONE && v0 != q.first_vector)) lane.load(pre, a.x, 0);
                    if (!ONE && v0 != q.first_vector) {
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
                    if (a.activation == kGroupNormSilu) forward_apply<T, VEC, true, store_of(MODE), B>(a, lane, pre, mean, scale, shift);
                    else forward_apply<T, VEC, false, store_of(MODE), B>(a, lane, pre, mean, scale, shift);
                }
                v0 += a.slice_vectors;
            } while (!ONE && v0 < q.end_vector);
        }
        if constexpr (!ONE) __syncthreads();
        n += gridDim.z;
    } while (!ONE && n < a.batch);
}

// Adds up the chunks' sums of four groups of a sample and leaves what the last launch reads: forward the
// statistics, backward the two means.
template<bool BACKWARD>
__global__ __launch_bounds__(256) void group_norm_finish(GnArgs a) {
    __shared__ double2 lds[256];
    const int in_slab = (int)(blockIdx.x * 4 + threadIdx.x % 4), g = (int)blockIdx.y * a.slab_groups + in_slab;
    const bool on = in_slab < a.slab_groups && g < a.groups;
    for (long long n = blockIdx.z; n < a.batch; n += gridDim.z) {
        double2 t = {0, 0};
        if (on) {
            const double2* part = (const double2*)a.group_part + (n * gridDim.y + blockIdx.y) * a.chunks * a.slab_groups + in_slab;
            for (int k = (int)threadIdx.x / 4; k < a.chunks; k += 8 * 64) {
                double2 in[8];
                #pragma unroll
                for (int u = 0; u < 8; u++) in[u] = part[(long long)min(k + u * 64, a.chunks - 1) * a.slab_groups];
                #pragma unroll
                for (int u = 0; u < 8; u++) {
                    t.x += k + u * 64 < a.chunks ? in[u].x : 0.0;
                    t.y += k + u * 64 < a.chunks ? in[u].y : 0.0;
                }
            }
        }
        lds[threadIdx.x] = t;
        for (int half = 128; half >= 4; half /= 2) {
            __syncthreads();
            if ((int)threadIdx.x < half) {
                lds[threadIdx.x].x += lds[threadIdx.x + half].x;
                lds[threadIdx.x].y += lds[threadIdx.x + half].y;
            }
        }
        if (threadIdx.x < 4 && on) {
            t = lds[threadIdx.x];
            float* to = (BACKWARD ? a.means : a.stats) + (n * a.groups + g) * 2;
            if constexpr (BACKWARD) {
                to[0] = (float)(t.x * a.inv_count);
                to[1] = (float)(t.y * a.inv_count);
            } else {
                write_stats(to, t.x * a.inv_count, t.y * a.inv_count, a.eps);
            }
        }
        __syncthreads();
    }
}

// ---- backward ----------------------------------------------------------------------------------

constexpr int backward_batch(int) { return 2; }                               // pixels of both arrays

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
    float mean[VEC], scale[VEC], shift[VEC], rstd[VEC];
    __device__ __forceinline__ void load(const GnArgs& a, const Place& q, long long n, int v) {
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
__device__ __forceinline__ void backward_lane_sums(const GnArgs& a, const Lane<T, VEC>& lane, const Channels<T, VEC>& ch,
                                                   Vec<T, VEC> (&x)[B], Vec<T, VEC> (&g)[B],
                                                   float (&s1)[VEC], float (&s2)[VEC]) {
    typedef Vec<T, VEC> V;
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
    #pragma unroll 1
    for (; i + 2 * B <= lane.whole; i += B) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            add(x[u], g[u]);
            x[u] = lane.load(a.x, i + B + u);
            g[u] = lane.load(a.dout, i + B + u);
            in_order();
        }
    }
    #pragma unroll 1
    for (; i < lane.runs; i += B) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            if (i + u < lane.count) add(x[u], g[u]);
            if (i + B + u < lane.runs) {
                x[u] = lane.load(a.x, i + B + u);
                g[u] = lane.load(a.dout, i + B + u);
            }
        }
    }
    #pragma unroll
    for (int j = 0; j < VEC; j++) s2[j] *= ch.rstd[j];
}

// Adds the lanes' sums up to channels (for the gradients of weight and bias, into `row` of the workspace) and
// those, weighted, to the slab's groups.
template<typename T, int VEC, int MODE, bool ONE>
__device__ __forceinline__ void backward_group_sums(const GnArgs& a, const Place& q, long long n, int v0, bool on, const float (&s1)[VEC], const float (&s2)[VEC],
                                                    float weight, double* lds, double (*sums)[2], float (*stat)[2], long long row, bool add_to_row) {
    const int slice_channels = a.slice_vectors * VEC;
    const int c0 = v0 * VEC, here = min(v0 + a.slice_vectors, q.end_vector) * VEC - c0;      // channels of the slice
    float* lanes = (float*)lds;                                   // [which][row][channel of the slice]
    double* totals = lds + a.rows * slice_channels;               // [which][channel]
    double2* partial = (double2*)(lds + gn_pairs_at(a.rows, slice_channels));                // [part][channel]
    float* to = a.channel_part + row * 2 * a.channels + c0;
    if (q.ty < a.rows) {
        float* at = lanes + q.ty * slice_channels + q.tx * VEC;
        #pragma unroll
        for (int j = 0; j < VEC; j++) {
            at[j] = on ? s1[j] : 0.0f;
            at[a.rows * slice_channels + j] = on ? s2[j] : 0.0f;
        }
    }
    __syncthreads();
    auto add_rows = [&](int c, int first, int step) {
        double2 t = {0, 0};
        #pragma unroll 4
        for (int r = first; r < a.rows; r += step) {
            t.x += lanes[r * slice_channels + c];
            t.y += lanes[(a.rows + r) * slice_channels + c];
        }
        return t;
    };
    // VEC rows of threads are as many as there are channels: each such part adds some of the rows up (8 samples of
    // 256 pixels of 1280 channels, backward: 14.4 us, 15.9 with one thread to a channel)
    const int parts = a.rows / VEC;
    if (parts > 1) {
        if (q.ty < parts * VEC) {
            const int c = q.ty % VEC * a.slice_vectors + q.tx, part = q.ty / VEC;
            partial[part * slice_channels + c] = add_rows(c, part, parts);
        }
        __syncthreads();
    }
    for (int c = (int)threadIdx.x; c < here; c += (int)blockDim.x) {
        float w[1] = {weight};
        if (!ONE || c != (int)threadIdx.x) load_params<T, 1>(w, a.weight, a.weight_fp32, c0 + c, 1.0f);
        double t1 = 0, t2 = 0;
        if (parts > 1) {
            #pragma unroll 4
            for (int i = 0; i < parts; i++) {
                t1 += partial[i * slice_channels + c].x;
                t2 += partial[i * slice_channels + c].y;
            }
        } else {
            const double2 t = add_rows(c, 0, 1);
            t1 = t.x;
            t2 = t.y;
        }
        to[c] = add_to_row ? to[c] + (float)t1 : (float)t1;
        to[a.channels + c] = add_to_row ? to[a.channels + c] + (float)t2 : (float)t2;
        totals[c] = t1 * w[0];
        totals[slice_channels + c] = t2 * w[0];
    }
    __syncthreads();
    const int per = 1 << a.per_group_log2, start = c0 - q.first_vector * VEC;                // channels of the slab
    const int first = (int)threadIdx.x >> a.per_group_log2, part = (int)threadIdx.x & (per - 1), step = (int)blockDim.x >> a.per_group_log2;
    for (int base = 0; base < q.groups; base += step) {
        const int at = base + first;
        const int lo = max(at * a.group_channels, start), hi = min((at + 1) * a.group_channels, start + here);
        double t1 = 0, t2 = 0;
        if (at < q.groups) {
            #pragma unroll 2
            for (int c = lo + part; c < hi; c += per) {
                t1 += totals[c - start];
                t2 += totals[slice_channels + c - start];
            }
        }
        t1 = add_over(t1, a.per_group_log2);
        t2 = add_over(t2, a.per_group_log2);
        if (at < q.groups && part == 0) {
            if constexpr (!ONE) {
                sums[at][0] += t1;
                sums[at][1] += t2;
            } else if constexpr (MODE == kSums) {
                ((double2*)a.group_part)[((n * gridDim.y + q.slab) * a.chunks + q.chunk) * a.slab_groups + at] = {t1, t2};
            } else {
                stat[at][0] = (float)(t1 * a.inv_count);
                stat[at][1] = (float)(t2 * a.inv_count);
            }
        }
    }
    __syncthreads();
}

// dx = rstd (w dz - c1 - h c2) as dz scale - (x - mean) e - d
template<typename T, int VEC, bool SILU, int STORE, int B>
__device__ __forceinline__ void backward_apply(const GnArgs& a, const Place& q, const Lane<T, VEC>& lane, const Channels<T, VEC>& ch,
                                               Vec<T, VEC> (&x)[B], Vec<T, VEC> (&g)[B], float (*stat)[2]) {
    typedef Vec<T, VEC> V;
    float d[VEC], e[VEC];
    int gr[VEC];
    groups_of<VEC>(gr, a, q, lane.v);
    #pragma unroll
    for (int j = 0; j < VEC; j++) {
        e[j] = ch.rstd[j] * ch.rstd[j] * stat[gr[j]][1];
        d[j] = ch.rstd[j] * stat[gr[j]][0];
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
    #pragma unroll 1
    for (; i + 2 * B <= lane.whole; i += B) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            lane.template store<STORE>(a.out, i + u, one(x[u], g[u]));
            x[u] = lane.load(a.x, i + B + u);
            g[u] = lane.load(a.dout, i + B + u);
            in_order();
        }
    }
    #pragma unroll 1
    for (; i < lane.runs; i += B) {
        #pragma unroll
        for (int u = 0; u < B; u++) {
            if (i + u < lane.count) lane.template store<STORE>(a.out, i + u, one(x[u], g[u]));
            if (i + B + u < lane.runs) {
                x[u] = lane.load(a.x, i + B + u);
                g[u] = lane.load(a.dout, i + B + u);
            }
        }
    }
}

// dw and db: the channels' sums added over the rows of the workspace, 16 channels to a workgroup.
template<typename T>
__device__ __forceinline__ void add_params(const GnArgs& a, int block, double* lds) {
    constexpr int W = kGroupNormParamChannels;
    const int tx = (int)threadIdx.x % W, ty = (int)threadIdx.x / W, rows = (int)blockDim.x / W;
    const int c = block * W + tx;
    double2* lanes = (double2*)lds;
    double2 t = {0, 0};
    if (c < a.channels) {
        const float* part = a.channel_part + c;
        for (long long r = ty; r < a.channel_rows; r += 8 * rows) {
            float in[8], in2[8];                                  // eight at a time, so that they are waited for once
            #pragma unroll
            for (int u = 0; u < 8; u++) {
                const float* at = part + min(r + u * rows, a.channel_rows - 1) * 2 * a.channels;
                in[u] = at[0];
                in2[u] = at[a.channels];
            }
            #pragma unroll
            for (int u = 0; u < 8; u++) {
                const bool on = r + u * rows < a.channel_rows;
                t.x += on ? in[u] : 0.0f;
                t.y += on ? in2[u] : 0.0f;
            }
        }
    }
    lanes[threadIdx.x] = t;
    __syncthreads();
    if (ty == 0 && c < a.channels) {
        #pragma unroll 4
        for (int i = 1; i < rows; i++) {
            t.x += lanes[i * W + tx].x;
            t.y += lanes[i * W + tx].y;
        }
        store_param<T>(a.dbias, a.weight_fp32, c, (float)t.x);
        store_param<T>(a.dweight, a.weight_fp32, c, (float)t.y);
    }
}

template<typename T, int VEC, int MODE, bool ONE>
__global__ __launch_bounds__(kGroupNormMaxThreads, 4) void group_norm_backward(GnArgs a) {
    extern __shared__ __attribute__((aligned(16))) double lds[];
    __shared__ double sums[kGroupNormMaxSlabGroups][2];
    __shared__ __attribute__((aligned(8))) float stat[kGroupNormMaxSlabGroups][2];
    if (applies_only(MODE) && (int)blockIdx.x < a.param_x) {          // a part of the grid that comes first
        const long long block = ((long long)blockIdx.z * gridDim.y + blockIdx.y) * a.param_x + blockIdx.x;
        if (block < a.param_blocks) add_params<T>(a, (int)block, lds);
        return;
    }
    const Place q = place_of<does_both(MODE)>(a, (int)blockIdx.x - (applies_only(MODE) ? a.param_x : 0));
    const bool silu = a.activation == kGroupNormSilu;
    long long n = q.n;
    do {
        constexpr int B = backward_batch(MODE);
        constexpr bool KEEP = ONE && does_both(MODE);             // what a lane needs of its channels, from the sums on
        Vec<T, VEC> px[B], pg[B];
        Channels<T, VEC> ch;
        float weight[1] = {1.0f};                                 // of the channel that this thread adds up
        const bool kept = ONE || applies_only(MODE) || q.end_vector - q.first_vector <= a.slice_vectors;
        {
            const Lane<T, VEC> lane(a, q, n, q.first_vector);
            if (lane.count) {
                lane.load(px, a.x, 0);
                lane.load(pg, a.dout, 0);
                if constexpr (KEEP) ch.load(a, q, n, lane.v);
            }
        }
        if constexpr (!applies_only(MODE)) {
            if constexpr (ONE) {
                const int c = q.first_vector * VEC + (int)threadIdx.x;
                if (c < a.channels) load_params<T, 1>(weight, a.weight, a.weight_fp32, c, 1.0f);
            } else {
                clear_sums(q, sums);
            }
            int v0 = q.first_vector;
            do {
                const Lane<T, VEC> lane(a, q, n, v0);
                float s1[VEC], s2[VEC];
                if (lane.count) {
                    if (!ONE && v0 != q.first_vector) {
                        lane.load(px, a.x, 0);
                        lane.load(pg, a.dout, 0);
                    }
                    if constexpr (!KEEP) ch.load(a, q, n, lane.v);
                    auto sum = [&](Vec<T, VEC> (&x)[B], Vec<T, VEC> (&g)[B]) {
                        if (silu) backward_lane_sums<T, VEC, true, B>(a, lane, ch, x, g, s1, s2);
                        else backward_lane_sums<T, VEC, false, B>(a, lane, ch, x, g, s1, s2);
                    };
                    if constexpr (does_both(MODE)) {
                        Vec<T, VEC> x[B], g[B];                   // `px` and `pg` stay, to be applied
                        #pragma unroll
                        for (int u = 0; u < B; u++) { x[u] = px[u]; g[u] = pg[u]; }
                        sum(x, g);
                    } else {
                        sum(px, pg);
                    }
                }
                backward_group_sums<T, VEC, MODE, ONE>(a, q, n, v0, lane.count != 0, s1, s2, weight[0], lds, sums, stat, q.n * a.chunks + q.chunk, n != q.n);
                v0 += a.slice_vectors;
            } while (!ONE && v0 < q.end_vector);
        }
        if constexpr (MODE == kSums) {
            if constexpr (!ONE) write_part(a, q, n, sums);
        } else {
            if (applies_only(MODE) && a.finish) {
                load_stats(a.means, a, q, n, stat);
            } else if constexpr (applies_only(MODE) || !ONE) {
                if constexpr (applies_only(MODE)) gather_chunks(a, q, n, lds, sums);
                for (int g = (int)threadIdx.x; g < q.groups; g += (int)blockDim.x) {
                    stat[g][0] = (float)(sums[g][0] * a.inv_count);
                    stat[g][1] = (float)(sums[g][1] * a.inv_count);
                }
                __syncthreads();
            }
            int v0 = q.first_vector;
            do {
                const Lane<T, VEC> lane(a, q, n, v0);
                if (lane.count) {
                    if (!kept || (!ONE && v0 != q.first_vector)) {
                        lane.load(px, a.x, 0);
                        lane.load(pg, a.dout, 0);
                    }
                    if constexpr (!KEEP) ch.load(a, q, n, lane.v);
                    if (silu) backward_apply<T, VEC, true, store_of(MODE), B>(a, q, lane, ch, px, pg, stat);
                    else backward_apply<T, VEC, false, store_of(MODE), B>(a, q, lane, ch, px, pg, stat);
                }
                v0 += a.slice_vectors;
            } while (!ONE && v0 < q.end_vector);
        }
        if constexpr (!ONE) __syncthreads();
        n += gridDim.z;
    } while (!ONE && n < a.batch);
}

template<typename T>
__global__ __launch_bounds__(256) void group_norm_params(GnArgs a) {
    __shared__ __attribute__((aligned(16))) double lds[256 * 2];
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
    a.batch = c.batch; a.pixels = c.pixels; a.channel_rows = p.channel_rows;
    a.inv_count = 1.0 / ((double)c.pixels * (double)p.group_channels);
    a.inv_group_channels = 1.0f / (float)p.group_channels; a.eps = c.eps;
    a.gather_groups = p.slab_groups < p.threads ? p.slab_groups : p.threads;
    a.gather_threads = p.threads / a.gather_groups;
    a.inv_slice = ((1u << 20) + p.slice_vectors - 1) / p.slice_vectors;
    a.inv_gather = ((1u << 20) + a.gather_groups - 1) / a.gather_groups;
    a.channels = c.channels; a.groups = c.groups; a.group_channels = p.group_channels; a.row_vectors = p.row_vectors;
    a.slab_vectors = p.slab_vectors; a.slab_groups = p.slab_groups; a.slice_vectors = p.slice_vectors;
    a.rows = p.rows; a.chunks = p.chunks;
    const long long runs = gn_ceil(c.pixels, p.rows);
    a.runs = (int)(runs / p.chunks);
    a.more_runs = (int)(runs % p.chunks);
    a.last_pixels = (int)(c.pixels % p.rows);
    a.last_chunk = a.last_pixels ? (int)((runs - 1) % p.chunks) : -1;
    while (a.per_group_log2 < 6 && (p.slab_groups << (a.per_group_log2 + 1)) <= p.threads) a.per_group_log2++;
    a.weight_fp32 = c.weight_fp32; a.activation = c.activation; a.finish = p.finish;
    a.straddle = p.group_channels % p.vec != 0;
    a.passes = gn_sum_passes(p.vec, p.group_channels);
    return a;
}

dim3 grid_of(const GroupNormPlan& p) { return dim3((unsigned)p.chunks, (unsigned)p.slabs, (unsigned)p.batch_blocks); }
dim3 finish_grid_of(const GroupNormPlan& p) { return dim3((unsigned)(p.slab_groups + 3) / 4, (unsigned)p.slabs, (unsigned)p.batch_blocks); }

template<typename T, int VEC, int KIND>
hipError_t forward_of(const GroupNormCall& c, hipStream_t stream) {
    const GroupNormPlan& p = c.plan;
    const GnArgs a = args_of(c);
    const dim3 grid = grid_of(p), block((unsigned)p.threads);
    if (p.chunks == 1) {
        if (p.merge) group_norm_forward<T, VEC, kBothMerge, KIND><<<grid, block, p.lds_bytes, stream>>>(a);
        else group_norm_forward<T, VEC, kBoth, KIND><<<grid, block, p.lds_bytes, stream>>>(a);
        return hipGetLastError();
    }
    group_norm_forward<T, VEC, kSums, KIND><<<grid, block, p.lds_bytes, stream>>>(a);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    if (p.finish) {
        group_norm_finish<false><<<finish_grid_of(p), dim3(256), 0, stream>>>(a);
        err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    if (p.stream) group_norm_forward<T, VEC, kApplyStream, KIND == kLoops ? kLoops : kOne><<<grid, block, p.lds_bytes, stream>>>(a);
    else group_norm_forward<T, VEC, kApply, KIND == kLoops ? kLoops : kOne><<<grid, block, p.lds_bytes, stream>>>(a);
    return hipGetLastError();
}

template<typename T, int VEC, bool ONE>
hipError_t backward_of(const GroupNormCall& c, hipStream_t stream) {
    const GroupNormPlan& p = c.plan;
    GnArgs a = args_of(c);
    dim3 grid = grid_of(p);
    const dim3 block((unsigned)p.threads);
    const bool params = c.dweight || c.dbias;
    if (p.chunks == 1) {
        if (p.merge) group_norm_backward<T, VEC, kBothMerge, ONE><<<grid, block, p.lds_bytes, stream>>>(a);
        else group_norm_backward<T, VEC, kBoth, ONE><<<grid, block, p.lds_bytes, stream>>>(a);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess || !params) return err;
        group_norm_params<T><<<dim3((unsigned)p.param_blocks), dim3(256), 0, stream>>>(a);
        return hipGetLastError();
    }
    group_norm_backward<T, VEC, kSums, ONE><<<grid, block, p.lds_bytes, stream>>>(a);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    if (p.finish) {
        group_norm_finish<true><<<finish_grid_of(p), dim3(256), 0, stream>>>(a);
        err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    if (params) {
        a.param_blocks = p.param_blocks;
        a.param_x = p.param_x;
        grid.x += (unsigned)a.param_x;
    }
    if (p.stream) group_norm_backward<T, VEC, kApplyStream, ONE><<<grid, block, p.lds_bytes, stream>>>(a);
    else group_norm_backward<T, VEC, kApply, ONE><<<grid, block, p.lds_bytes, stream>>>(a);
    return hipGetLastError();
}

template<typename T, int VEC>
hipError_t launch_of(const GroupNormCall& c, bool backward, hipStream_t stream) {
    // (instantiated for full vectors only: the others are built once, with the loops)
    if constexpr (sizeof(T) * VEC == 16) {
        if (c.plan.batch_blocks == c.batch && c.plan.slab_vectors <= c.plan.slice_vectors) {
            if (backward) return backward_of<T, VEC, true>(c, stream);
            return c.plan.group_channels >= VEC ? forward_of<T, VEC, kOneWide>(c, stream) : forward_of<T, VEC, kOne>(c, stream);
        }
    }
    return backward ? backward_of<T, VEC, false>(c, stream) : forward_of<T, VEC, kLoops>(c, stream);
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
