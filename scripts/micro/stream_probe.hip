// Streaming-read policy probe (round 6): which load shape / cache policy / grid reads N bytes ONCE fastest on gfx950?
//   hipcc --offload-arch=gfx950 -Xclang -target-feature -Xclang -packed-fp32-ops -O3 -o stream_probe scripts/micro/stream_probe.hip && ./stream_probe [bytes]
// Variants: plain 16-byte loads with U loads in flight per lane, the same non-temporal, LDS-DMA (global_load_lds, 1 KiB per
// wave-instruction) with aux = 0 / 2 (nt) and R pieces in flight per wave; grids of CUs x {1, 2, 4, 8} workgroups of 256.
// Prints one line per variant: us per pass and TB/s.  A micro-benchmark, not part of any library.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include <hip/hip_runtime.h>

#define CK(x) do { hipError_t e_ = (x); if (e_ != hipSuccess) { std::fprintf(stderr, "%s: %s\n", #x, hipGetErrorString(e_)); std::exit(1); } } while (0)

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int U, bool kNt>
__global__ __launch_bounds__(256) void k_plain(const u32x4* __restrict__ src, uint64_t n16, uint32_t* __restrict__ sink) {
    uint32_t acc = 0;
    const uint64_t stride = uint64_t(gridDim.x) * 256;
    uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x;
    for (; i + (U - 1) * stride < n16; i += U * stride) {
        u32x4 v[U];
#pragma unroll
        for (int k = 0; k < U; k++) v[k] = kNt ? __builtin_nontemporal_load(src + i + k * stride) : src[i + k * stride];
#pragma unroll
        for (int k = 0; k < U; k++) acc ^= v[k].x ^ v[k].y ^ v[k].z ^ v[k].w;
    }
    for (; i < n16; i += stride) { const u32x4 a = src[i]; acc ^= a.x ^ a.y ^ a.z ^ a.w; }
    if (acc == 0x9E3779B9u) sink[blockIdx.x] = acc;
}

// contiguous variant: a workgroup owns a contiguous span, a wave reads U x 1 KiB consecutive pieces per step
template <int U, bool kNt>
__global__ __launch_bounds__(256) void k_span(const u32x4* __restrict__ src, uint64_t n16, uint32_t* __restrict__ sink) {
    uint32_t acc = 0;
    const uint64_t waves = uint64_t(gridDim.x) * 4;
    const uint64_t wave = uint64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const uint64_t per = ((n16 / 64 + waves - 1) / waves) * 64;  // 16-byte units per wave (multiple of 64); the last waves get less
    const uint64_t begin = wave * per, end = begin + per < n16 ? begin + per : n16;
    if (begin >= n16) return;
    const u32x4* p = src + begin + (threadIdx.x & 63);
    const uint64_t mine = end - begin;
    uint64_t i = 0;
    for (; i + uint64_t(U) * 64 <= mine; i += uint64_t(U) * 64) {
        u32x4 v[U];
#pragma unroll
        for (int k = 0; k < U; k++) v[k] = kNt ? __builtin_nontemporal_load(p + i + k * 64) : p[i + k * 64];
#pragma unroll
        for (int k = 0; k < U; k++) acc ^= v[k].x ^ v[k].y ^ v[k].z ^ v[k].w;
    }
    for (; i + (threadIdx.x & 63) < mine; i += 64) { const u32x4 a = kNt ? __builtin_nontemporal_load(p + i) : p[i]; acc ^= a.x ^ a.y ^ a.z ^ a.w; }
    if (acc == 0x9E3779B9u) sink[blockIdx.x] = acc;
}

// LDS-DMA: every wave keeps R pieces of 1 KiB in flight into its own LDS ring and "consumes" a piece with one ds_read
template <int R, int kAux>
__global__ __launch_bounds__(256) void k_glds(const uint8_t* __restrict__ src, uint64_t bytes, uint32_t* __restrict__ sink) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint8_t* ring = lds + size_t(w) * R * 1024;
    const uint64_t waves = uint64_t(gridDim.x) * 4;
    const uint64_t wave = uint64_t(blockIdx.x) * 4 + w;
    const uint64_t all = bytes / 1024, per = (all + waves - 1) / waves;
    const uint64_t first = wave * per;
    if (first >= all) return;
    const uint64_t pieces = first + per <= all ? per : all - first;
    const uint8_t* p = src + first * 1024 + size_t(lane) * 16;
    uint32_t acc = 0;
    auto issue = [&](uint64_t piece) {
        __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) void*>(reinterpret_cast<uintptr_t>(p + piece * 1024)),
                                         reinterpret_cast<__attribute__((address_space(3))) void*>(uint32_t(reinterpret_cast<uintptr_t>(ring + (piece % R) * 1024))),
                                         16, 0, kAux);
    };
    uint64_t issued = 0;
    for (; issued < uint64_t(R) && issued < pieces; issued++) issue(issued);
    for (uint64_t c = 0; c < pieces; c++) {
        // wait until piece c has landed: at most (issued - c - 1) DMAs may stay outstanding
        if (issued - c - 1 >= uint64_t(R - 1)) __builtin_amdgcn_s_waitcnt(0x0F70 | ((R - 1) & 0xF) | (((R - 1) >> 4) << 14));
        else __builtin_amdgcn_s_waitcnt(0x0F70);  // tail: vmcnt(0)
        acc ^= *reinterpret_cast<const uint32_t*>(ring + (c % R) * 1024 + lane * 4);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the slot is free again
        if (issued < pieces) { issue(issued); issued++; }
    }
    if (acc == 0x9E3779B9u) sink[blockIdx.x] = acc;
}

struct Variant { const char* name; void (*launch)(const uint8_t*, uint64_t, uint32_t*, int, hipStream_t); };

template <int U, bool kNt> void l_plain(const uint8_t* s, uint64_t b, uint32_t* k, int g, hipStream_t st) {
    hipLaunchKernelGGL((k_plain<U, kNt>), dim3(g), dim3(256), 0, st, reinterpret_cast<const u32x4*>(s), b / 16, k);
}
template <int U, bool kNt> void l_span(const uint8_t* s, uint64_t b, uint32_t* k, int g, hipStream_t st) {
    hipLaunchKernelGGL((k_span<U, kNt>), dim3(g), dim3(256), 0, st, reinterpret_cast<const u32x4*>(s), b / 16, k);
}
template <int R, int A> void l_glds(const uint8_t* s, uint64_t b, uint32_t* k, int g, hipStream_t st) {
    hipLaunchKernelGGL((k_glds<R, A>), dim3(g), dim3(256), 4 * R * 1024, st, s, b, k);
}

int main(int argc, char** argv) {
    const uint64_t bytes = argc > 1 ? std::strtoull(argv[1], nullptr, 10) : 788ull * 1000 * 1000;
    const uint64_t flush_bytes = 1ull << 30;
    uint8_t *d = nullptr, *f = nullptr;
    CK(hipMalloc(reinterpret_cast<void**>(&d), bytes + (1 << 20)));
    CK(hipMalloc(reinterpret_cast<void**>(&f), flush_bytes + (1 << 20)));
    CK(hipMemset(d, 1, bytes + (1 << 20)));
    CK(hipMemset(f, 2, flush_bytes + (1 << 20)));
    uint32_t* sink = reinterpret_cast<uint32_t*>(d + bytes);
    uint32_t* fsink = reinterpret_cast<uint32_t*>(f + flush_bytes);
    hipDeviceProp_t prop;
    CK(hipGetDeviceProperties(&prop, 0));
    const int cus = prop.multiProcessorCount;
    hipEvent_t e0, e1;
    CK(hipEventCreate(&e0));
    CK(hipEventCreate(&e1));
    const Variant vs[] = {
        {"plain  U=4", l_plain<4, false>}, {"plain  U=8", l_plain<8, false>}, {"plain  U=16", l_plain<16, false>},
        {"nt     U=4", l_plain<4, true>},  {"nt     U=8", l_plain<8, true>},  {"nt     U=16", l_plain<16, true>},
        {"span   U=4", l_span<4, false>},  {"span   U=8", l_span<8, false>},  {"span nt U=4", l_span<4, true>}, {"span nt U=8", l_span<8, true>},
        {"glds a0 R=4", l_glds<4, 0>}, {"glds a0 R=8", l_glds<8, 0>}, {"glds a0 R=16", l_glds<16, 0>},
        {"glds nt R=4", l_glds<4, 2>}, {"glds nt R=8", l_glds<8, 2>}, {"glds nt R=16", l_glds<16, 2>},
    };
    const int mults[] = {1, 2, 4, 8, 16};
    std::printf("device %s, %d CUs, %.1f MB per pass (cold = 1 GiB flush read before every pass)\n", prop.name, cus, bytes / 1e6);
    for (const Variant& v : vs) {
        for (int m : mults) {
            const int grid = cus * m;
            if (v.launch == l_glds<16, 0> || v.launch == l_glds<16, 2>) { if (m > 2) continue; }  // 64 KiB of LDS per workgroup
            if ((v.launch == l_glds<8, 0> || v.launch == l_glds<8, 2>) && m > 4) continue;
            double hot = 0, cold = 0;
            for (int pass = 0; pass < 2; pass++) {
                double sum = 0;
                const int iters = 10;
                for (int i = -2; i < iters; i++) {
                    if (pass == 1) l_plain<4, false>(f, flush_bytes, fsink, 4096, nullptr);
                    CK(hipEventRecord(e0, nullptr));
                    v.launch(d, bytes, sink, grid, nullptr);
                    CK(hipEventRecord(e1, nullptr));
                    CK(hipEventSynchronize(e1));
                    float ms = 0;
                    CK(hipEventElapsedTime(&ms, e0, e1));
                    if (i >= 0) sum += double(ms) * 1000.0;
                }
                (pass == 0 ? hot : cold) = sum / iters;
            }
            std::printf("%-14s grid %5d (x%-2d): hot %8.1f us %5.2f TB/s | cold %8.1f us %5.2f TB/s\n", v.name, grid, m, hot, bytes / hot / 1e6,
                        cold, bytes / cold / 1e6);
            std::fflush(stdout);
        }
    }
    return 0;
}
