// Group norm with an activation over (batch, pixels, channels) arrays whose channels lie last: how the work
// is cut (plain C++, shared with the CPU tests) and the launch functions (group_norm.hip).
//
// Vocabulary:
//   vector   `vec` channels of one pixel, 16 bytes at most: the widest power of two that divides the row
//   slab     consecutive whole groups of channels, a whole number of vectors: one workgroup's share of a row
//   slice    the part of a slab a workgroup walks at a time, one vector per lane (nearly always all of it)
//   rows     pixels a workgroup works on side by side, next to each other: a run
//   chunk    one workgroup's share of a sample's pixels: chunk k of K takes runs k, k + K, ..., so that all
//            workgroups together move through memory as one window (512x512 pixels of 256 channels: 77.7 us; with
//            a contiguous piece for each, 79.4)
#pragma once

#include <cstddef>
#include <cstdint>

namespace sideaware {

enum GroupNormType { kGroupNormFp32 = 0, kGroupNormBf16 = 1, kGroupNormFp16 = 2 };
enum GroupNormActivation { kGroupNormNone = 0, kGroupNormSilu = 1 };

struct GroupNormPlan {
    int vec = 1;                    // channels per vector
    int row_vectors = 0;            // vectors per pixel
    int group_channels = 0;
    int slab_vectors = 0, slabs = 0;
    int slab_groups = 0;            // groups of a (full) slab
    int slice_vectors = 0;          // vectors of a slice: lanes side by side
    int rows = 1;
    int threads = 64;
    int chunks = 1;                 // per sample; 1: sums and application in one launch
    long long batch_blocks = 1;     // one launch: workgroups share out the samples of a slab, sample n to n % batch_blocks
    size_t lds_bytes = 0;
    // Chunks: whether a launch of its own adds up their sums, instead of every workgroup that applies them.
    bool finish = false;
    // workspace: doubles of the groups' sums [sample][slab][chunk][group of slab][2]; backward, with a launch
    // that adds them up, floats of the groups' means [sample][group][2]; backward, floats of the channels' sums
    // [row][2][channel], a row for each (sample or batch block, chunk)
    size_t group_part_bytes = 0, means_bytes = 0;
    long long channel_rows = 0;
    size_t workspace_bytes = 0;
    bool stream = false;            // the arrays do not fit the Infinity Cache together, with a quarter to spare
    bool merge = false;             // one launch: slabs are no whole memory lines, which the L2 puts together
    long long blocks = 0;           // workgroups of a launch over the array: chunks x slabs x batch_blocks
    int param_blocks = 0;           // workgroups that add up the channels' sums
    int param_x = 0;                // chunks: by how many they widen the second launch's first axis
    bool ok = false;
};

// Two workgroups of eight waves to a CU, which leaves each lane 128 registers (one to a CU: 103 us instead of 79 for
// 512x512 pixels of 256 channels).
constexpr int kGroupNormMaxThreads = 512;
constexpr int kGroupNormMaxSliceChannels = 1024;  // of lanes' sums in LDS
constexpr int kGroupNormMaxSlabGroups = 256;
constexpr int kGroupNormParamChannels = 16;       // channels per workgroup that adds up their sums
constexpr long long kGroupNormMaxLanePixels = 256;         // that a lane adds in fp32 before its sums become doubles
// A sample's part of the smallest slab that one launch takes: at 20 KiB (2 samples of 256 pixels of 1280 channels) one
// launch takes 8 us and two take 17, at 80 KiB (2 of 1024 pixels of 640 channels) one takes 15 and two take 11.
constexpr long long kGroupNormOneLaunchBytes = 32 << 10;
// Several times that is still read a second time out of the L2s, if all that run at once hold no more than this (the
// L2s hold half of it; 16 samples of 1024 pixels of 640 channels, 20 MiB: 15.3 us, two launches 18.2; backward, 40 MiB, 26.6
// and 29.8; 48 samples, backward, 80 MiB: 86 and 69), every CU has a workgroup and their pieces of a row are half a
// memory line or more (64 samples of 1024 pixels of 512 channels: pieces of 64 bytes 31.5, of 32 bytes 77, two launches 36.5).
constexpr long long kGroupNormHeldBytes = 64 << 20;
constexpr int kGroupNormPieceBytes = 64, kGroupNormLineBytes = 128;
// Where the arrays exceed the Infinity Cache, pieces are whole lines (256 samples of 256 pixels of 1280 channels: pieces of 80
// bytes 211 us, two launches 103); arrays up to this size are read in whatever pieces.
constexpr long long kGroupNormPiecesBytes = 8 << 20;
// What every workgroup of the second launch may read to add up the chunks' sums by itself: 64 KiB (4 samples of 16384
// pixels of 128 channels) 20.6 us, 21.7 with a launch between; 256 KiB (65536 pixels of 512 channels) 44.3 and 42.6.
constexpr long long kGroupNormGatherBytes = 64 << 10;
constexpr long long kGroupNormCacheBytes = 256ll << 20;    // the Infinity Cache
constexpr long long kGroupNormMaxGrid = 65535;            // of the second and third axis
constexpr long long kGroupNormMaxRowsBytes = 1ll << 30;    // a lane's offset among the rows has 32 bits

inline long long gn_ceil(long long a, long long b) { return (a + b - 1) / b; }

// The most groups that one vector's channels belong to.  Vectors start d, 2d, ... channels into a group, d being the
// greatest common divisor of the two lengths; one that starts at a group's last d has the most, those d channels and
// vec - d more: 3 for a vector of 8 and groups of 5 (1 + 5 + 2 channels), 1 where groups are whole vectors.
constexpr int gn_groups_of_vector(int vec, int group_channels) {
    int d = vec, rest = group_channels;
    while (rest) {
        const int next = d % rest;
        d = rest;
        rest = next;
    }
    return 1 + (vec - d + group_channels - 1) / group_channels;
}
// How often the lanes' sums go through LDS, two groups of every vector at a time.
constexpr int gn_sum_passes(int vec, int group_channels) { return (gn_groups_of_vector(vec, group_channels) + 1) / 2; }
// Backward, where in LDS the pairs of doubles of the parts of the rows lie, in doubles: behind two floats for each lane's
// channel and two doubles for each channel of the slice, on a pair's boundary (7 channels, 73 rows: 525 doubles come first).
constexpr int gn_pairs_at(int rows, int slice_channels) { return ((rows + 2) * slice_channels + 1) / 2 * 2; }

inline GroupNormPlan plan_group_norm(long long batch, long long pixels, int channels, int groups, int element_bytes, bool backward,
                                     int num_cus, long long cache_bytes = kGroupNormCacheBytes) {
    GroupNormPlan p;
    if (batch < 1 || pixels < 1 || channels < 1 || groups < 1 || channels % groups || num_cus < 1) return p;
    p.vec = 16 / element_bytes;
    while (channels % p.vec) p.vec /= 2;
    p.row_vectors = channels / p.vec;
    p.group_channels = channels / groups;
    // the smallest slab: whole groups and whole vectors (both divide the row, so it does too)
    int unit = p.group_channels;
    while (unit % p.vec) unit += p.group_channels;
    const int unit_vectors = unit / p.vec, unit_groups = unit / p.group_channels, units = channels / unit;

    const long long row_bytes = (long long)channels * element_bytes;
    if (row_bytes > kGroupNormMaxRowsBytes || pixels > 0x7fffffffll) return p;

    int most_slice = kGroupNormMaxSliceChannels / p.vec;
    if (most_slice > kGroupNormMaxThreads) most_slice = kGroupNormMaxThreads;
    auto cut = [&](int m) {                        // slabs of m units
        p.slab_vectors = m * unit_vectors;
        p.slab_groups = m * unit_groups;
        p.slabs = (int)gn_ceil(units, m);
        p.slice_vectors = p.slab_vectors < most_slice ? p.slab_vectors : most_slice;
        const long long most_rows = kGroupNormMaxThreads / p.slice_vectors;
        p.rows = (int)(pixels < most_rows ? pixels : most_rows);
        while (p.rows > 1 && p.rows * row_bytes > kGroupNormMaxRowsBytes) p.rows /= 2;
    };
    // the widest slabs: of one slice, if a unit is not wider; all of about the same width
    int most_units = kGroupNormMaxSlabGroups / unit_groups;
    if (most_units > most_slice / unit_vectors) most_units = most_slice / unit_vectors > 1 ? most_slice / unit_vectors : 1;
    most_units = (int)gn_ceil(units, gn_ceil(units, most_units));

    // One launch where a sample's part of the smallest slab is little, or the L2s hold the parts of all workgroups that run
    // at once: they then read it a second time out of the caches.  Else the pixels are cut into chunks as well, and a second launch applies
    // what the first one summed.
    const long long unit_bytes = pixels * unit_vectors * p.vec * element_bytes, piece_bytes = unit_vectors * p.vec * element_bytes;
    // wider slabs while there are workgroups enough without, up to 512 bytes of a row
    int m = 1;
    while (2 * m <= most_units && 2 * m * unit_vectors <= 32 && batch * gn_ceil(units, 2 * m) >= 2 * num_cus &&
           2 * m * unit_bytes <= kGroupNormOneLaunchBytes)
        m *= 2;
    const long long array_bytes = batch * pixels * row_bytes, all_bytes = array_bytes * (backward ? 3 : 2);
    // (how the work is cut, and with it the workspace, does not depend on what a user tunes)
    const bool beyond = all_bytes > kGroupNormCacheBytes / 4 * 3;
    p.stream = all_bytes > cache_bytes / 4 * 3;
    bool one = unit_bytes <= kGroupNormOneLaunchBytes &&
               (m * piece_bytes >= (beyond ? kGroupNormLineBytes : kGroupNormPieceBytes) || m == units || array_bytes <= kGroupNormPiecesBytes);
    if (!one && !beyond) {
        m = (int)gn_ceil(kGroupNormPieceBytes, piece_bytes);
        if (m > units) m = units;
        const long long all = batch * gn_ceil(units, m), at_once = all < 2 * num_cus ? all : 2 * num_cus;
        one = m <= most_units && all >= num_cus && at_once * m * unit_bytes * (backward ? 2 : 1) <= kGroupNormHeldBytes;
        const int slice = m * unit_vectors < most_slice ? m * unit_vectors : most_slice;
        one = one && gn_ceil(pixels, kGroupNormMaxThreads / slice) <= kGroupNormMaxLanePixels;
    }
    if (one) {
        cut(m);
        p.merge = p.slabs > 1 && (long long)p.slab_vectors * p.vec * element_bytes % kGroupNormLineBytes != 0;
        const long long want = gn_ceil(4ll * num_cus, p.slabs);
        p.batch_blocks = batch < want ? batch : want;
    } else {
        cut(most_units);
        const long long step = p.rows;
        // no more workgroups than the device holds at once, unless the (sample, slab) pairs are more already, and at least
        // four pixels a lane.  From half as many pairs on each has one chunk, so places stay empty, and behind a full turn a
        // nearly empty one may run: forward, 257 samples of 4096 pixels of 320 channels 449 us, 256 samples 391; 513 821, 512 765
        const long long want = 2ll * num_cus / (batch * p.slabs), most = gn_ceil(pixels, 4 * step);
        const long long least = gn_ceil(pixels, step * kGroupNormMaxLanePixels);
        long long k = want < most ? want : most;
        if (k < least) k = least;
        p.chunks = (int)(k < 1 ? 1 : k);
        p.finish = (long long)p.chunks * p.slab_groups * 16 > kGroupNormGatherBytes;
        p.batch_blocks = batch < kGroupNormMaxGrid ? batch : kGroupNormMaxGrid;
    }
    const int lanes = p.slice_vectors * p.rows;
    p.threads = (lanes + 63) / 64 * 64;
    // forward: four doubles a lane.  backward: two floats for each lane and channel, two doubles for each channel
    // of the slice, then two doubles for each part of the rows and channel.  Either: two doubles a thread where the chunks'
    // sums are added.
    const int slice_channels = p.slice_vectors * p.vec;
    const size_t sums = backward ? gn_pairs_at(p.rows, slice_channels) * sizeof(double) + (size_t)(p.rows / p.vec) * slice_channels * 2 * sizeof(double)
                                 : (size_t)lanes * 4 * sizeof(double);
    const size_t gather = (size_t)p.threads * 2 * sizeof(double);
    p.lds_bytes = sums > gather ? sums : gather;
    p.blocks = p.batch_blocks * p.slabs * p.chunks;
    p.group_part_bytes = p.chunks > 1 ? (size_t)(batch * p.slabs * p.chunks) * p.slab_groups * 2 * sizeof(double) : 0;
    p.channel_rows = backward ? p.batch_blocks * p.chunks : 0;
    p.param_blocks = backward ? (int)gn_ceil(channels, kGroupNormParamChannels) : 0;
    p.means_bytes = backward && p.finish ? ((size_t)batch * groups * 2 * sizeof(float) + 15) / 16 * 16 : 0;
    p.workspace_bytes = p.group_part_bytes + p.means_bytes + (size_t)p.channel_rows * 2 * channels * sizeof(float);
    // the workgroups that add up the parameters' gradients widen the first axis, for each of the others: by a multiple of
    // eight where it is long, so that the XCD that summed a chunk up applies it as well, out of its L2 if that holds it
    // (4 samples of 16384 pixels of 128 channels: 24.9 us, 26.1 without)
    const long long others = p.slabs * p.batch_blocks;
    long long param_x = gn_ceil(p.param_blocks, others);
    if (p.chunks >= 16) param_x = (param_x + 7) / 8 * 8;
    p.param_x = (int)param_x;
    p.ok = p.slabs <= kGroupNormMaxGrid && (p.chunks + param_x) * others <= 0x7fffffffll && p.lds_bytes <= (56u << 10);
    return p;
}

struct GroupNormCall {
    GroupNormPlan plan;
    long long batch = 0, pixels = 0;
    int channels = 0, groups = 0;
    int type = 0;                   // GroupNormType of x, out, dout, dx
    bool weight_fp32 = false;       // of weight, bias and their gradients; otherwise the arrays' type
    int activation = 0;
    float eps = 0;
    const void* x = nullptr;
    const void* dout = nullptr;     // backward
    const void* weight = nullptr;   // null: 1
    const void* bias = nullptr;     // null: 0
    float* stats = nullptr;         // (batch, groups, 2): mean and 1/sqrt(var + eps); written forward, read backward
    void* out = nullptr;            // y, or dx
    void* dweight = nullptr;        // backward; may be null
    void* dbias = nullptr;
    void* workspace = nullptr;
};

// Enqueue the launches on `stream` of the current device; a hipError_t.
int launch_group_norm_forward(const GroupNormCall& call, void* stream);
int launch_group_norm_backward(const GroupNormCall& call, void* stream);

}  // namespace sideaware
