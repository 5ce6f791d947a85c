// Reads "batch pixels channels groups element_bytes backward" lines and checks what the kernels rely on of
// group_norm.h's plan: every (sample, pixel, channel) belongs to one workgroup and lane, groups are whole
// inside slabs, and every workgroup's accesses to LDS and to the workspace stay inside what the plan asks for.
#include <cstdio>
#include <vector>

#include "../../l2_torch_alloc_amd/csrc/group_norm.h"

using namespace sideaware;

#define REQUIRE(x) do { if (!(x)) { std::printf("FAIL %s: %s", #x, line); return 1; } } while (0)

int main() {
    char line[256];
    long long batch, pixels;
    int channels, groups, element, backward, cases = 0, one = 0;
    while (std::fgets(line, sizeof line, stdin)) {
        if (std::sscanf(line, "%lld %lld %d %d %d %d", &batch, &pixels, &channels, &groups, &element, &backward) != 6) continue;
        cases++;
        const GroupNormPlan p = plan_group_norm(batch, pixels, channels, groups, element, backward, 256);
        REQUIRE(p.ok);
        REQUIRE(p.vec >= 1 && p.vec * element <= 16 && channels % p.vec == 0 && p.row_vectors * p.vec == channels);
        REQUIRE(p.group_channels * groups == channels);
        // slabs: whole vectors, whole groups, all of the row
        REQUIRE(p.slabs >= 1 && (long long)p.slabs * p.slab_vectors >= p.row_vectors && (long long)(p.slabs - 1) * p.slab_vectors < p.row_vectors);
        REQUIRE(p.slab_vectors * p.vec == p.slab_groups * p.group_channels);
        REQUIRE(p.slab_groups >= 1 && p.slab_groups <= kGroupNormMaxSlabGroups);
        REQUIRE(p.slice_vectors >= 1 && p.slice_vectors * p.vec <= kGroupNormMaxSliceChannels && p.slice_vectors <= p.slab_vectors);
        // lanes
        REQUIRE(p.rows >= 1 && p.rows <= pixels && p.slice_vectors * p.rows <= p.threads);
        REQUIRE(p.threads % 64 == 0 && p.threads >= 64 && p.threads <= kGroupNormMaxThreads);
        // chunks: none empty, none with more pixels to a lane than its sums may hold
        REQUIRE(p.chunks >= 1 && (long long)(p.chunks - 1) * p.rows < pixels && (long long)p.chunks * p.rows < (1ll << 32));
        REQUIRE((pixels + (long long)p.chunks * p.rows - 1) / ((long long)p.chunks * p.rows) <= kGroupNormMaxLanePixels);
        REQUIRE((long long)p.rows * channels * element <= kGroupNormMaxRowsBytes);
        // samples
        const long long samples = p.batch_blocks;
        REQUIRE(samples >= 1 && samples <= batch && samples <= 65535 && p.slabs <= 65535 && p.blocks == samples * p.slabs * p.chunks);
        const long long others = p.slabs * samples;
        REQUIRE((p.chunks + (p.param_blocks + others - 1) / others) * others <= 0x7fffffffll);
        REQUIRE((long long)p.param_x * others >= p.param_blocks && (p.chunks + (long long)p.param_x) * others <= 0x7fffffffll);
        // thread numbers are divided by multiplying with 2^20 / slice_vectors
        for (int t = 0; t < p.threads; t++) {
            const unsigned inv = ((1u << 20) + p.slice_vectors - 1) / p.slice_vectors;
            REQUIRE((int)((t * inv) >> 20) == t / p.slice_vectors);
            const int gather = p.slab_groups < p.threads ? p.slab_groups : p.threads;
            const unsigned inv_gather = ((1u << 20) + gather - 1) / gather;
            REQUIRE((int)((t * inv_gather) >> 20) == t / gather);
        }
        // ... and channels of a slab by the fp32 reciprocal of a group's, one step of correction either way
        for (int g = 0; g <= p.slab_groups; g++) {
            for (int d = -1; d <= 1; d++) {
                const long long c = (long long)g * p.group_channels + d;
                if (c < 0 || c >= (long long)p.slab_vectors * p.vec) continue;
                const int guess = (int)((float)(int)c * (1.0f / (float)p.group_channels));
                REQUIRE(guess - (int)(c / p.group_channels) <= 1 && (int)(c / p.group_channels) - guess <= 1);
            }
        }
        // LDS: forward four doubles a lane; backward two floats for each lane's channel, and two
        // doubles for each channel of the slice; two doubles a thread
        const size_t slice_channels = (size_t)p.slice_vectors * p.vec;
        if (backward) REQUIRE(p.lds_bytes >= p.rows * slice_channels * 8 + 2 * slice_channels * 8);
        // (and where rows are many, two doubles for each channel and part of the rows)
        if (backward) REQUIRE(p.lds_bytes >= (p.rows + 2) * slice_channels * 8 + (p.rows / p.vec) * slice_channels * 16);
        if (!backward) REQUIRE(p.lds_bytes >= (size_t)p.slice_vectors * p.rows * 32);
        REQUIRE(p.lds_bytes >= (size_t)p.threads * 16);
        REQUIRE(p.lds_bytes + kGroupNormMaxSlabGroups * 24 <= 65536);
        // workspace
        if (p.chunks > 1) {
            const long long last = (((batch - 1) * p.slabs + p.slabs - 1) * p.chunks + p.chunks - 1) * p.slab_groups * 2 + (p.slab_groups - 1) * 2 + 1;
            REQUIRE((size_t)(last + 1) * 8 <= p.group_part_bytes);
            if (p.finish && backward) REQUIRE(p.means_bytes >= (size_t)batch * groups * 8 && p.means_bytes % 16 == 0);
        } else {
            REQUIRE(p.group_part_bytes == 0);
            one++;
        }
        if (backward) {
            REQUIRE(p.channel_rows == samples * p.chunks);
            REQUIRE(p.workspace_bytes == p.group_part_bytes + p.means_bytes + (size_t)p.channel_rows * 2 * channels * 4);
            REQUIRE((long long)p.param_blocks * kGroupNormParamChannels >= channels);
        } else {
            REQUIRE(p.workspace_bytes == p.group_part_bytes);
        }
    }
    std::printf("cases=%d one_launch=%d ok\n", cases, one);
    return 0;
}
