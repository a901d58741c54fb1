// kv8.cuh -- what the writer, the reader and the attention of the 8-bit key/value cache share.
//
// k_cache, v_cache: [n_blocks][Hkv][block_size][D] e4m3 codes, so the tokens of one (block, head)
// are block_size * D contiguous bytes; k_scale, v_scale: [n_blocks][Hkv] fp32, powers of two
// 2^e with -40 <= e <= 40.  The value is code * scale.
//
// Why powers of two: e4m3 is a floating-point format, so a finer scale would not make its
// relative rounding error (2^-4) smaller, and a power of two keeps every step around the codes
// exact: x / scale has one rounding (to the code), a block whose scale grows keeps its old
// codes' values (only those that become subnormal are rounded again), code * scale is exact in
// bf16 and fp32, and the attention can carry the scale of V in the exponent of its weights.
#pragma once

#include <atomic>

#include "common.cuh"

namespace b200 {

constexpr int kKv8MaxExp = 40;
constexpr float kKv8MinScale = 9.094947017729282e-13f;  // 2^-40
constexpr float kKv8MaxScale = 1099511627776.f;         // 2^40

// The smallest scale 2^e in range with amax <= 448 * 2^e; amax finite and not negative.
// amax = (1 + m / 2^23) 2^x and 448 = 1.75 * 2^8, so e = x - 8, or x - 7 where 1 + m / 2^23 > 1.75.
__device__ __forceinline__ float kv8_scale_for(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(-kKv8MaxExp, min(kKv8MaxExp, e));
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Four values -> four codes (a in the lowest byte): nearest even, |x| > 448 becomes 448, NaN stays NaN.
__device__ __forceinline__ uint32_t kv8_encode4(float a, float b, float c, float d) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}

// Four codes -> four fp16 values, the lower two in `lo` (exact: every e4m3 value is an fp16 value).
__device__ __forceinline__ void kv8_decode4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(codes));
}

// log2 of the block sizes that are built (16, 32, 64, 128 tokens), else -1.
inline int kv8_log2_block(int block_size) {
    for (int s = 4; s <= 7; ++s)
        if (block_size == 1 << s) return s;
    return -1;
}

// Sizes shared by the three entries.
inline int kv8_check_cache(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                           const int* block_table, int B, int max_blocks, int n_blocks, int block_size, int Hkv,
                           int D) {
    if (!k_cache || !v_cache || !k_scale || !v_scale || !block_table) return B200LAB_ERR_INVALID;
    if (B < 1 || max_blocks < 1 || n_blocks < 1 || block_size < 1 || Hkv < 1 || D < 1) return B200LAB_ERR_INVALID;
    if ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) return B200LAB_ERR_INVALID;
    if (kv8_log2_block(block_size) < 0 || (D != 64 && D != 128 && D != 256)) return B200LAB_ERR_UNSUPPORTED;
    if ((long long)n_blocks * Hkv > 0x7fffffffLL) return B200LAB_ERR_UNSUPPORTED;
    // positions and lengths are 32-bit
    if ((long long)max_blocks * block_size > 0x40000000LL) return B200LAB_ERR_UNSUPPORTED;
    return B200LAB_OK;
}

// What the launches need to know of the current device, asked of the runtime once a device: its
// ordinal (-1 on an error), whether it is an sm_100 part, its SMs.
struct Kv8Device {
    int ordinal, sms;
    int status;
};
inline Kv8Device kv8_device() {
    constexpr int kMost = 64;
    static std::atomic<int> seen[kMost];  // 0: not asked yet, else 2 * SMs + (an sm_100 part)
    Kv8Device d = {-1, 0, B200LAB_ERR_CUDA};
    if (cudaGetDevice(&d.ordinal) != cudaSuccess) return d;
    int v = d.ordinal < kMost ? seen[d.ordinal].load(std::memory_order_relaxed) : 0;
    if (v == 0) {
        const int rc = check_device_sm100();
        if (rc == B200LAB_ERR_CUDA) return d;
        v = 2 * device_sm_count() + (rc == B200LAB_OK);
        if (d.ordinal < kMost) seen[d.ordinal].store(v, std::memory_order_relaxed);
    }
    d.sms = v >> 1;
    d.status = (v & 1) ? B200LAB_OK : B200LAB_ERR_DEVICE;
    return d;
}

// Launches `kern` with programmatic stream serialisation: every kernel of this cache waits
// (grid_dependency_wait) before it touches memory and then lets the next one be scheduled, so
// the steps append -> attend -> ... of a decode loop follow one another without the launch gap.
// `cluster`: CTAs of a cluster.
template <typename Kern, typename... Args>
int kv8_launch_clusters(int cluster, Kern kern, dim3 grid, int threads, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    // The launch's own status alone: the thread's last error may be an earlier call's, and a call that reported it
    // would have written the cache, or stopped between its two kernels.
    if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) {
        (void)cudaGetLastError();  // it is reported here, and not again by the program's next check
        return B200LAB_ERR_CUDA;
    }
    count_launch(1);
    return B200LAB_OK;
}
template <typename Kern, typename... Args>
int kv8_launch(Kern kern, dim3 grid, int threads, size_t smem, cudaStream_t st, Args... args) {
    return kv8_launch_clusters(1, kern, grid, threads, smem, st, args...);
}

}  // namespace b200
