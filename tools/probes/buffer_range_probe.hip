// Probe (tools/probes): the range check of raw buffer loads on gfx950 where part of the offset is scalar.  A load returns zeros where
// lane offset + scalar offset + size reaches beyond num_records (dword by dword for 16-byte loads), also where the scalar offset alone is at or
// beyond it.  Every address lies inside the 256 KiB allocation whatever the check does.
//   hipcc --offload-arch=gfx950 -O3 -Xclang -target-feature -Xclang -packed-fp32-ops -o tools/probes/buffer_range_probe.bin \
//         tools/probes/buffer_range_probe.hip && tools/probes/buffer_range_probe.bin
#include <hip/hip_runtime.h>
#include <cstdio>
#include <vector>
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
__global__ void probe(const unsigned* p, unsigned* o, int num_records, int soff) {
    auto r = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, num_records, 0x00020000);
    const int t = threadIdx.x;
    const u32x4 near = __builtin_amdgcn_raw_buffer_load_b128(r, t * 16, soff, 0), far = __builtin_amdgcn_raw_buffer_load_b128(r, t * 16 + 2048, soff, 0);
    o[t] = near[0]; o[64 + t] = near[3]; o[128 + t] = far[0];
    o[192 + t] = __builtin_amdgcn_raw_buffer_load_b8(r, t, soff, 0);
    o[256 + t] = __builtin_amdgcn_raw_buffer_load_b32(r, t * 4, soff, 0);
    o[320 + t] = __builtin_amdgcn_raw_buffer_load_b16(r, t * 2, soff, 0);
}
int main() {
    const int N = 1 << 16;
    std::vector<unsigned> h(N), got(384);
    for (int i = 0; i < N; ++i) h[i] = 0x01000193u * (i + 1) | 0x01010101u;          // (no byte is zero)
    unsigned *p, *o;
    if (hipMalloc(&p, N * 4) != hipSuccess || hipMalloc(&o, 384 * 4) != hipSuccess) return 1;
    if (hipMemcpy(p, h.data(), N * 4, hipMemcpyHostToDevice) != hipSuccess) return 1;
    int failed = 0;
    for (auto& c : std::vector<std::pair<int, int>>{{4096, 0}, {512, 0}, {1024, 512}, {520, 16}, {48, 32}, {4096, 2048}, {100, 60},       // scalar offset inside
                                                     {512, 512}, {0, 0},                                                              // at the end
                                                     {512, 1024}, {512, 16384}, {0, 256}, {100, 65536}}) {                            // beyond it
        const int n = c.first, soff = c.second;
        hipLaunchKernelGGL(probe, dim3(1), dim3(64), 0, 0, p, o, n, soff);
        if (hipMemcpy(got.data(), o, 384 * 4, hipMemcpyDeviceToHost) != hipSuccess) return 1;
        auto want = [&](int off, int size) {
            unsigned w = 0;
            if (off + soff + size <= n) __builtin_memcpy(&w, (const char*)h.data() + off + soff, size);
            return w;
        };
        int bad = 0;
        for (int t = 0; t < 64; ++t)
            bad += (got[t] != want(t * 16, 4)) + (got[64 + t] != want(t * 16 + 12, 4)) + (got[128 + t] != want(t * 16 + 2048, 4)) + (got[192 + t] != want(t, 1)) +
                   (got[256 + t] != want(t * 4, 4)) + (got[320 + t] != want(t * 2, 2));
        printf("num_records %5d, scalar offset %5d: %s (%d of 384 loads differ)\n", n, soff, bad ? "NOT as stated" : "as stated", bad);
        failed += bad != 0;
    }
    return failed != 0;
}
