// Appended after group_norm.hip: reads cases from the standard input and runs each through the file's own launch code.
//
//   backward batch pixels channels groups fp32 activation weight_fp32 cus in out
//
// `in`: x, weight, bias and, backward, dout and stats, one behind the other; `out`: the outputs, likewise (forward y and stats,
// backward dx, dweight and dbias).  fp32 or bf16.  Every array is a block of its own of exactly the bytes it needs.
#include <cstdio>

struct CpuArray {
    char* data = nullptr;
    size_t size;
    explicit CpuArray(size_t bytes) : size(bytes) {
        if (posix_memalign((void**)&data, 16, bytes ? bytes : 1) != 0) std::abort();
        std::memset(data, 0xff, bytes);
    }
    ~CpuArray() { std::free(data); }
    void read(FILE* f) { if (std::fread(data, 1, size, f) != size) std::abort(); }
    void write(FILE* f) { if (std::fwrite(data, 1, size, f) != size) std::abort(); }
};

int main() {
    using namespace sideaware;
    int backward, channels, groups, fp32, activation, weight_fp32, cus;
    long long batch, pixels;
    char in[1024], out[1024];
    while (std::scanf("%d %lld %lld %d %d %d %d %d %d %1023s %1023s", &backward, &batch, &pixels, &channels, &groups, &fp32, &activation, &weight_fp32,
                      &cus, in, out) == 11) {
        GroupNormCall call;
        call.plan = plan_group_norm(batch, pixels, channels, groups, fp32 ? 4 : 2, backward != 0, cus);
        if (!call.plan.ok) return 3;
        const size_t bytes = (size_t)(batch * pixels * channels) * (fp32 ? 4 : 2), param = (size_t)channels * (fp32 || weight_fp32 ? 4 : 2);
        CpuArray x(bytes), w(param), b(param), dout(backward ? bytes : 0), stats((size_t)batch * groups * 8), y(bytes), dw(param), db(param),
            ws(call.plan.workspace_bytes);
        FILE* f = std::fopen(in, "rb");
        if (!f) return 4;
        x.read(f);
        w.read(f);
        b.read(f);
        if (backward) {
            dout.read(f);
            stats.read(f);
        }
        std::fclose(f);
        call.batch = batch; call.pixels = pixels; call.channels = channels; call.groups = groups;
        call.weight_fp32 = fp32 || weight_fp32; call.activation = activation; call.eps = 1e-5f;
        call.x = x.data; call.weight = w.data; call.bias = b.data; call.stats = (float*)stats.data; call.out = y.data; call.workspace = ws.data;
        if (backward) {
            call.dout = dout.data; call.dweight = dw.data; call.dbias = db.data;
        }
        cpu_launches = cpu_chunked = 0;
        if ((fp32 ? launch_vec<float>(call, backward != 0, nullptr) : launch_vec<__bf16>(call, backward != 0, nullptr)) != hipSuccess) return 5;
        f = std::fopen(out, "wb");
        if (!f) return 6;
        y.write(f);
        if (backward) {
            dw.write(f);
            db.write(f);
        } else {
            stats.write(f);
        }
        std::fclose(f);
        std::printf("launches=%ld chunked=%ld\n", cpu_launches, cpu_chunked);
        std::fflush(stdout);
    }
    return 0;
}
