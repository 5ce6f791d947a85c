// Appended after the kernel template: runs one launch on the CPU, lane by lane, over arrays read from
// files, and writes the output back.  Lanes run one after another, so ops that exchange values between
// lanes cannot be run this way.
//
//   argv: grid num_bytes base_offset stripe_log2 val in0 in1 in2 in3 mem out0   ("-": no such array)
//
// Every array is a posix_memalign block of exactly the bytes it needs, shifted by base_offset (in0, in1
// of the same width and out0 together), under AddressSanitizer.
#include <cstdio>
#include <cstdlib>
#include <string>
#include <vector>

#include "../../l2_torch_alloc_amd/csrc/launch_plan.h"

struct Block {
    char* block = nullptr;
    char* data = nullptr;
    size_t size = 0;
    void make(size_t off, size_t bytes) {
        if (posix_memalign((void**)&block, 2u << 20, off + bytes + (bytes == 0)) != 0) std::abort();
        std::memset(block, 0xAB, off);
        data = block + off;
        size = bytes;
    }
    ~Block() { std::free(block); }
    void read(const char* path, size_t off) {
        if (std::string(path) == "-") return;
        FILE* f = std::fopen(path, "rb");
        if (!f) std::abort();
        std::fseek(f, 0, SEEK_END);
        make(off, (size_t)std::ftell(f));
        std::rewind(f);
        if (std::fread(data, 1, size, f) != size) std::abort();
        std::fclose(f);
    }
};

int main(int argc, char** argv) {
    if (argc != 12) return 2;
    const unsigned grid = (unsigned)std::atoi(argv[1]);
    const size_t num_bytes = (size_t)std::atoll(argv[2]), off = (size_t)std::atoll(argv[3]);
    const unsigned stripe_log2 = (unsigned)std::atoi(argv[4]);
    const int val = (int)std::atoll(argv[5]);
    Block in[4], mem, out;
    in[0].read(argv[6], off);
    in[1].read(argv[7], sizeof(vi1) == sizeof(vi0) && !sa_inputs_gathered ? off : 0);
    in[2].read(argv[8], 0);
    in[3].read(argv[9], 0);
    mem.read(argv[10], 0);
    out.make(off, num_bytes);
    std::memset(out.data, 0xCD, num_bytes);

    const long long nv = (long long)(num_bytes / 16);
    const int element = 16 / vec_size, ragged = (int)(num_bytes % 16) / element;
    const unsigned long long base = sideaware_kernel_meta[2] ? (unsigned long long)out.data : (unsigned long long)in[0].data;
    sideaware::LaunchPlan p;
    if (sa_sided) {
        sideaware::SideMap side;
        side.pair_mask = SA_SIDE_PAIR_MASK;
        side.dealing = 3;
        p = sideaware::plan_launch_sided(base, nv, sideaware_kernel_meta[0], SA_NUM_XCD, stripe_log2 % 9, 1, grid / SA_NUM_XCD, side,
                                         (unsigned)sa_followed_vector_bytes);
    } else {
        p = sideaware::plan_launch(base, nv, sideaware_kernel_meta[0], SA_NUM_XCD, 1ull << stripe_log2, 1, grid / SA_NUM_XCD);
    }
    if (ragged && p.tail_block < 0) p.tail_block = 0;
    gridDim = {p.grid, 1, 1};
    blockDim = {SA_WG_THREADS, 1, 1};
    for (unsigned b = 0; b < p.grid; b++) {
        for (unsigned t = 0; t < SA_WG_THREADS; t++) {
            blockIdx = {b, 0, 0};
            threadIdx = {t, 0, 0};
            KERNEL_NAME((size_type)nv, (size_type)p.full_tiles, (size_type)p.b0, (size_type)p.u_count, (size_type)p.run, p.r_word, p.grid,
                        val, (const vi0*)in[0].data, (vo0*)out.data, nullptr, p.tail_block, nullptr, nullptr, nullptr,
                        (const vi1*)in[1].data, (const vi2*)in[2].data, (const vi3*)in[3].data, (int*)mem.data
#ifdef RAGGED_TAIL
                        , ragged
#endif
            );
        }
    }
    for (size_t i = 0; i < off; i++) if ((unsigned char)out.block[i] != 0xAB) return 3;
    FILE* f = std::fopen(argv[11], "wb");
    if (!f || std::fwrite(out.data, 1, num_bytes, f) != num_bytes) return 4;
    std::fclose(f);
    return 0;
}
