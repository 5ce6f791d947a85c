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
    float* channel_part;
    long long batch, pixels, chunk_pixels, batch_blocks, channel_rows, main_blocks;
    double inv_count;               // 1 / (pixels * channels of a group)
    int channels, groups, group_channels, row_vectors;
    int slab_vectors, slabs, slab_groups, slice_vectors, rows, chunks;
    int weight_fp32, activation;
    float eps;
};

template<typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
    T v[VEC];
};

template<typename T>
__device__ __forceinline__ float load_param(const void* p, int fp32, int c, float missing) {
    if (!p) return missing;
    return fp32 ? ((const float*)p)[c] : (float)((const T*)p)[c];
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

// Where this workgroup works and which vector of the row and which pixels this lane has.
struct Place {
    long long n;                    // sample (its first, where a workgroup has several)
    int slab, chunk;
    int first_vector, end_vector;   // of the slab
    int first_group, groups;        // of the slab
    long long p0, p1;               // pixels of the chunk
    int tx, ty;
};

__device__ __forceinline__ Place place_of(const GnArgs& a, long long block) {
    Place q;
    q.chunk = (int)(block % a.chunks);
    const long long rest = block / a.chunks;
    q.slab = (int)(rest % a.slabs);
    q.n = rest / a.slabs;
    q.first_vector = q.slab * a.slab_vectors;
    q.end_vector = min(q.first_vector + a.slab_vectors, a.row_vectors);
    q.first_group = q.slab * a.slab_groups;
    q.groups = min(a.slab_groups, a.groups - q.first_group);
    q.p0 = q.chunk * a.chunk_pixels;
    q.p1 = min(q.p0 + a.chunk_pixels, a.pixels);
    q.ty = (int)threadIdx.x / a.slice_vectors;
    q.tx = (int)threadIdx.x - q.ty * a.slice_vectors;
    return q;
}

// Adds one double per (row, channel) of the lanes over the rows: the rows of the upper half hand theirs to
// the lower half until one row is left.  Every thread of the workgroup calls; `lane_on` says which have values.
template<int VEC>
__device__ __forceinline__ void add_rows(double (&s)[VEC], const GnArgs& a, const Place& q, bool lane_on, double* lds) {
    for (int left = a.rows; left > 1;) {
        const int half = (left + 1) / 2;
        if (lane_on && q.ty >= half && q.ty < left) {
            #pragma unroll
            for (int j = 0; j < VEC; j++) lds[((q.ty - half) * VEC + j) * a.slice_vectors + q.tx] = s[j];
        }
        __syncthreads();
        if (lane_on && q.ty < left - half) {
            #pragma unroll
            for (int j = 0; j < VEC; j++) s[j] += lds[(q.ty * VEC + j) * a.slice_vectors + q.tx];
        }
        __syncthreads();
        left = half;
    }
}

// Adds the channels' sums of row 0 up to the groups of the slab, into sums[group][which].
template<int VEC>
__device__ __forceinline__ void add_channels(const double (&s)[VEC], const GnArgs& a, const Place& q, int v0, bool lane_on, double* lds,
                                             double (*sums)[2], int which) {
    if (lane_on && q.ty == 0) {
        #pragma unroll
        for (int j = 0; j < VEC; j++) lds[q.tx * VEC + j] = s[j];
    }
    __syncthreads();
    const int c0 = v0 * VEC, c1 = min(v0 + a.slice_vectors, q.end_vector) * VEC;     // channels of the slice
    // a power of two of threads for every group, all in one wave
    int per = 1;
    while (per < 64 && per * 2 * q.groups <= (int)blockDim.x) per *= 2;
    const int first = (int)threadIdx.x / per, part = (int)threadIdx.x % per, step = (int)blockDim.x / per;
    for (int base = 0; base < q.groups; base += step) {
        const int g = base + first;
        const int lo = max((q.first_group + g) * a.group_channels, c0), hi = min((q.first_group + g + 1) * a.group_channels, c1);
        double t = 0;
        if (g < q.groups) {
            for (int c = lo + part; c < hi; c += per) t += lds[c - c0];
        }
        for (int d = per / 2; d > 0; d /= 2) t += __shfl_xor(t, d, 64);
        if (g < q.groups && part == 0) sums[g][which] += t;
    }
    __syncthreads();
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

constexpr int kBatch = 4;           // pixels whose loads a lane has in flight

// ---- forward -----------------------------------------------------------------------------------

template<typename T, int VEC>
__device__ __forceinline__ void forward_sums(const GnArgs& a, const Place& q, long long n, double* lds, double (*sums)[2]) {
    typedef Vec<T, VEC> V;
    for (int v0 = q.first_vector; v0 < q.end_vector; v0 += a.slice_vectors) {
        const int v = v0 + q.tx;
        const bool lane_on = q.ty < a.rows && v < q.end_vector;
        double d1[VEC], d2[VEC];
        #pragma unroll
        for (int j = 0; j < VEC; j++) d1[j] = d2[j] = 0;
        if (lane_on && q.p0 + q.ty < q.p1) {
            const V* x = (const V*)a.x + (n * a.pixels + q.p0 + q.ty) * a.row_vectors + v;
            const long long step = (long long)a.rows * a.row_vectors;
            const int count = (int)((q.p1 - q.p0 - q.ty + a.rows - 1) / a.rows);
            float pivot[VEC], s1[VEC], s2[VEC];
            const V first = *x;
            #pragma unroll
            for (int j = 0; j < VEC; j++) { pivot[j] = (float)first.v[j]; s1[j] = s2[j] = 0; }
            int i = 0;
            for (; i + kBatch <= count; i += kBatch) {
                V in[kBatch];
                #pragma unroll
                for (int u = 0; u < kBatch; u++) in[u] = x[u * step];
                x += kBatch * step;
                #pragma unroll
                for (int u = 0; u < kBatch; u++) {
                    #pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const float d = (float)in[u].v[j] - pivot[j];
                        s1[j] += d;
                        s2[j] = fmaf(d, d, s2[j]);
                    }
                }
            }
            for (; i < count; i++) {
                const V in = *x;
                x += step;
                #pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const float d = (float)in.v[j] - pivot[j];
                    s1[j] += d;
                    s2[j] = fmaf(d, d, s2[j]);
                }
            }
            #pragma unroll
            for (int j = 0; j < VEC; j++) {
                const double p = pivot[j], m = count;
                d1[j] = s1[j] + m * p;
                d2[j] = s2[j] + p * (2.0 * s1[j] + m * p);
            }
        }
        add_rows<VEC>(d1, a, q, lane_on, lds);
        add_channels<VEC>(d1, a, q, v0, lane_on, lds, sums, 0);
        add_rows<VEC>(d2, a, q, lane_on, lds);
        add_channels<VEC>(d2, a, q, v0, lane_on, lds, sums, 1);
    }
}

// mean and 1/sqrt(var + eps) of the slab's groups from their sums
__device__ __forceinline__ void forward_stats(const GnArgs& a, const Place& q, long long n, double (*sums)[2], float (*stat)[2], bool write) {
    for (int g = (int)threadIdx.x; g < q.groups; g += (int)blockDim.x) {
        const double mean = sums[g][0] * a.inv_count;
        double var = sums[g][1] * a.inv_count - mean * mean;
        if (var < 0) var = 0;                                     // rounding; a NaN stays one
        const float m = (float)mean, r = (float)(1.0 / sqrt(var + (double)a.eps));
        stat[g][0] = m;
        stat[g][1] = r;
        if (write) {
            float* to = a.stats + (n * a.groups + q.first_group + g) * 2;
            to[0] = m;
            to[1] = r;
        }
    }
    __syncthreads();
}

template<typename T, int VEC, bool SILU>
__device__ __forceinline__ void forward_apply(const GnArgs& a, const Place& q, long long n, float (*stat)[2]) {
    typedef Vec<T, VEC> V;
    for (int v0 = q.first_vector; v0 < q.end_vector; v0 += a.slice_vectors) {
        const int v = v0 + q.tx;
        if (q.ty >= a.rows || v >= q.end_vector || q.p0 + q.ty >= q.p1) continue;
        float mean[VEC], scale[VEC], shift[VEC];
        #pragma unroll
        for (int j = 0; j < VEC; j++) {
            const int c = v * VEC + j, g = c / a.group_channels - q.first_group;
            mean[j] = stat[g][0];
            scale[j] = stat[g][1] * load_param<T>(a.weight, a.weight_fp32, c, 1.0f);
            shift[j] = load_param<T>(a.bias, a.weight_fp32, c, 0.0f);
        }
        const long long at = (n * a.pixels + q.p0 + q.ty) * a.row_vectors + v;
        const V* x = (const V*)a.x + at;
        V* y = (V*)a.out + at;
        const long long step = (long long)a.rows * a.row_vectors;
        const int count = (int)((q.p1 - q.p0 - q.ty + a.rows - 1) / a.rows);
        auto one = [&](const V& in) {
            V o;
            #pragma unroll
            for (int j = 0; j < VEC; j++) {
                const float z = fmaf((float)in.v[j] - mean[j], scale[j], shift[j]);
                o.v[j] = (T)(SILU ? z * sigmoid(z) : z);
            }
            return o;
        };
        int i = 0;
        for (; i + kBatch <= count; i += kBatch) {
            V in[kBatch];
            #pragma unroll
            for (int u = 0; u < kBatch; u++) in[u] = x[u * step];
            #pragma unroll
            for (int u = 0; u < kBatch; u++) y[u * step] = one(in[u]);
            x += kBatch * step;
            y += kBatch * step;
        }
        for (; i < count; i++) {
            *y = one(*x);
            x += step;
            y += step;
        }
    }
}

enum Mode { kSums, kApply, kBoth };

template<typename T, int VEC, int MODE>
__global__ __launch_bounds__(kGroupNormMaxThreads) void group_norm_forward(GnArgs a) {
    extern __shared__ double lds[];
    __shared__ double sums[kGroupNormMaxSlabGroups][2];
    __shared__ float stat[kGroupNormMaxSlabGroups][2];
    const Place q = place_of(a, blockIdx.x);
    for (long long n = q.n; n < a.batch; n += a.batch_blocks) {   // once, unless samples are shared out
        if constexpr (MODE != kApply) {
            clear_sums(q, sums);
            forward_sums<T, VEC>(a, q, n, lds, sums);
        }
        if constexpr (MODE == kSums) {
            write_part(a, q, sums);
            return;
        }
        if constexpr (MODE == kApply) gather_chunks(a, q, lds, sums);
        forward_stats(a, q, n, sums, stat, q.chunk == 0);
        if (a.activation == kGroupNormSilu) forward_apply<T, VEC, true>(a, q, n, stat);
        else forward_apply<T, VEC, false>(a, q, n, stat);
        __syncthreads();
    }
}

// ---- backward ----------------------------------------------------------------------------------

// What a lane needs of its channels to have z and dz of a value.
template<typename T, int VEC>
struct Channels {
    float mean[VEC], rstd[VEC], w[VEC], b[VEC];
    __device__ __forceinline__ void load(const GnArgs& a, long long n, int v) {
        #pragma unroll
        for (int j = 0; j < VEC; j++) {
            const int c = v * VEC + j;
            const float* s = a.stats + (n * a.groups + c / a.group_channels) * 2;
            mean[j] = s[0];
            rstd[j] = s[1];
            w[j] = load_param<T>(a.weight, a.weight_fp32, c, 1.0f);
            b[j] = load_param<T>(a.bias, a.weight_fp32, c, 0.0f);
        }
    }
};

template<bool SILU>
__device__ __forceinline__ float grad_of_z(float dout, float h, float w, float b) {
    if constexpr (!SILU) return dout;
    const float z = fmaf(h, w, b), s = sigmoid(z);
    return dout * (s * fmaf(z, 1.0f - s, 1.0f));
}

template<typename T, int VEC, bool SILU>
__device__ __forceinline__ void backward_sums(const GnArgs& a, const Place& q, long long n, double* lds, double (*sums)[2], long long row,
                                              bool add_to_row) {
    typedef Vec<T, VEC> V;
    for (int v0 = q.first_vector; v0 < q.end_vector; v0 += a.slice_vectors) {
        const int v = v0 + q.tx;
        const bool lane_on = q.ty < a.rows && v < q.end_vector;
        double d1[VEC], d2[VEC];
        #pragma unroll
        for (int j = 0; j < VEC; j++) d1[j] = d2[j] = 0;
        if (lane_on && q.p0 + q.ty < q.p1) {
            Channels<T, VEC> ch;
            ch.load(a, n, v);
            const long long at = (n * a.pixels + q.p0 + q.ty) * a.row_vectors + v;
            const V* x = (const V*)a.x + at;
            const V* dout = (const V*)a.dout + at;
            const long long step = (long long)a.rows * a.row_vectors;
            const int count = (int)((q.p1 - q.p0 - q.ty + a.rows - 1) / a.rows);
            float s1[VEC], s2[VEC];
            #pragma unroll
            for (int j = 0; j < VEC; j++) s1[j] = s2[j] = 0;
            auto one = [&](const V& in, const V& g) {
                #pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const float h = ((float)in.v[j] - ch.mean[j]) * ch.rstd[j];
                    const float dz = grad_of_z<SILU>((float)g.v[j], h, ch.w[j], ch.b[j]);
                    s1[j] += dz;
                    s2[j] = fmaf(dz, h, s2[j]);
                }
            };
            int i = 0;
            for (; i + 2 <= count; i += 2) {
                const V in0 = x[0], in1 = x[step], g0 = dout[0], g1 = dout[step];
                one(in0, g0);
                one(in1, g1);
                x += 2 * step;
                dout += 2 * step;
            }
            for (; i < count; i++) {
                one(*x, *dout);
                x += step;
                dout += step;
            }
            #pragma unroll
            for (int j = 0; j < VEC; j++) { d1[j] = s1[j]; d2[j] = s2[j]; }
        }
        add_rows<VEC>(d1, a, q, lane_on, lds);
        add_rows<VEC>(d2, a, q, lane_on, lds);
        // the channels' sums, for the gradients of weight and bias; then weighted, for the group's
        if (lane_on && q.ty == 0) {
            float* to = a.channel_part + row * 2 * a.channels + v * VEC;
            #pragma unroll
            for (int j = 0; j < VEC; j++) {
                const int c = v * VEC + j;
                if (add_to_row) {
                    to[j] += (float)d1[j];
                    to[a.channels + j] += (float)d2[j];
                } else {
                    to[j] = (float)d1[j];
                    to[a.channels + j] = (float)d2[j];
                }
                const double w = load_param<T>(a.weight, a.weight_fp32, c, 1.0f);
                d1[j] *= w;
                d2[j] *= w;
            }
        }
        add_channels<VEC>(d1, a, q, v0, lane_on, lds, sums, 0);
        add_channels<VEC>(d2, a, q, v0, lane_on, lds, sums, 1);
    }
}

template<typename T, int VEC, bool SILU>
__device__ __forceinline__ void backward_apply(const GnArgs& a, const Place& q, long long n, float (*stat)[2]) {
    typedef Vec<T, VEC> V;
    for (int v0 = q.first_vector; v0 < q.end_vector; v0 += a.slice_vectors) {
        const int v = v0 + q.tx;
        if (q.ty >= a.rows || v >= q.end_vector || q.p0 + q.ty >= q.p1) continue;
        Channels<T, VEC> ch;
        ch.load(a, n, v);
        float c1[VEC], c2[VEC];
        #pragma unroll
        for (int j = 0; j < VEC; j++) {
            const int g = (v * VEC + j) / a.group_channels - q.first_group;
            c1[j] = stat[g][0];
            c2[j] = stat[g][1];
        }
        const long long at = (n * a.pixels + q.p0 + q.ty) * a.row_vectors + v;
        const V* x = (const V*)a.x + at;
        const V* dout = (const V*)a.dout + at;
        V* dx = (V*)a.out + at;
        const long long step = (long long)a.rows * a.row_vectors;
        const int count = (int)((q.p1 - q.p0 - q.ty + a.rows - 1) / a.rows);
        auto one = [&](const V& in, const V& g) {
            V o;
            #pragma unroll
            for (int j = 0; j < VEC; j++) {
                const float h = ((float)in.v[j] - ch.mean[j]) * ch.rstd[j];
                const float dz = grad_of_z<SILU>((float)g.v[j], h, ch.w[j], ch.b[j]);
                o.v[j] = (T)(ch.rstd[j] * (fmaf(dz, ch.w[j], -c1[j]) - h * c2[j]));
            }
            return o;
        };
        int i = 0;
        for (; i + 2 <= count; i += 2) {
            const V in0 = x[0], in1 = x[step], g0 = dout[0], g1 = dout[step];
            dx[0] = one(in0, g0);
            dx[step] = one(in1, g1);
            x += 2 * step;
            dout += 2 * step;
            dx += 2 * step;
        }
        for (; i < count; i++) {
            *dx = one(*x, *dout);
            x += step;
            dout += step;
            dx += step;
        }
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
__global__ __launch_bounds__(kGroupNormMaxThreads) void group_norm_backward(GnArgs a) {
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
        if constexpr (MODE != kApply) {
            clear_sums(q, sums);
            const long long row = q.n * a.chunks + q.chunk;
            if (silu) backward_sums<T, VEC, true>(a, q, n, lds, sums, row, n != q.n);
            else backward_sums<T, VEC, false>(a, q, n, lds, sums, row, n != q.n);
        }
        if constexpr (MODE == kSums) {
            write_part(a, q, sums);
            return;
        }
        if constexpr (MODE == kApply) gather_chunks(a, q, lds, sums);
        for (int g = (int)threadIdx.x; g < q.groups; g += (int)blockDim.x) {
            stat[g][0] = (float)(sums[g][0] * a.inv_count);
            stat[g][1] = (float)(sums[g][1] * a.inv_count);
        }
        __syncthreads();
        if (silu) backward_apply<T, VEC, true>(a, q, n, stat);
        else backward_apply<T, VEC, false>(a, q, n, stat);
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
    a.channel_part = (float*)((char*)c.workspace + p.group_part_bytes);
    a.batch = c.batch; a.pixels = c.pixels; a.chunk_pixels = p.chunk_pixels; a.batch_blocks = p.batch_blocks;
    a.channel_rows = p.channel_rows; a.main_blocks = p.blocks;
    a.inv_count = 1.0 / ((double)c.pixels * (double)p.group_channels);
    a.channels = c.channels; a.groups = c.groups; a.group_channels = p.group_channels; a.row_vectors = p.row_vectors;
    a.slab_vectors = p.slab_vectors; a.slabs = p.slabs; a.slab_groups = p.slab_groups; a.slice_vectors = p.slice_vectors;
    a.rows = p.rows; a.chunks = p.chunks;
    a.weight_fp32 = c.weight_fp32; a.activation = c.activation; a.eps = c.eps;
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
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
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
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
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
