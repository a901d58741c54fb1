// kv8_cache.cu -- writing new tokens into the paged 8-bit key/value cache, and reading it back.
//
// No counterpart in the reference, which keeps K and V as dense 16-bit tensors
// (src/attn_sm75.cu:107-112).  Layout and number format: kv8.cuh.
#include "errwords.h"
#include "kv8.cuh"

namespace b200 {
namespace {

__device__ int g_err_kv8_cache = 0;

__device__ __forceinline__ void report_invalid() { atomicExch(&g_err_kv8_cache, B200LAB_ERR_INVALID); }

// 8 consecutive input values, as loaded.
template <typename T> struct Raw8 {
    uint4 a;
    __device__ __forceinline__ void load(const T* p) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ float get(int i) const { return Elem<T>::to_f(reinterpret_cast<const T*>(&a)[i]); }
};
template <> struct Raw8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = *reinterpret_cast<const float4*>(p);
        b = *reinterpret_cast<const float4*>(p + 4);
    }
    __device__ __forceinline__ float get(int i) const {
        return i < 4 ? reinterpret_cast<const float*>(&a)[i] : reinterpret_cast<const float*>(&b)[i - 4];
    }
};

struct AppendArgs {
    const void* x[2];          // K, V
    long long stride_t[2], stride_h[2];
    uint8_t* cache[2];
    float* scale[2];
    const int* table;
    const int* lens;
    const int* cu;
    int max_seqlen, total, B, max_blocks, n_blocks, log2P, Hkv, log2D, items_per_seq;  // blocks a sequence may touch
    long long items;
};

constexpr int kAppendVecs = 8;  // vectors of 8 values a thread holds

// One item = the new tokens of one sequence that fall into one block, of one head, of K or V.
// kThreads threads hold them in registers (each value is read once from memory), reduce their
// largest magnitude to the block's scale and write the codes.  A block begun by an earlier call
// keeps a larger old scale; where the new tokens need a larger one, its codes are rounded to it
// first.  Only slots below the sequence's length are written.
// Bound by memory for prompts and by latency (three dependent loads: offsets, block id, data)
// for a step of one token a sequence, where a warp an item keeps the grid to one short wave.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads < 128 ? 128 : kThreads, kThreads <= 128 && sizeof(T) == 2 ? 8 : 1)
    kv8_append_kernel(const AppendArgs a) {
    constexpr int kCta = kThreads < 128 ? 128 : kThreads;
    grid_dependency_wait();
    allow_dependent_launch();
    const int tid = threadIdx.x % kThreads;
    const long long item = (long long)blockIdx.x * (kCta / kThreads) + threadIdx.x / kThreads;
    if (item >= a.items) return;  // whole warps; whole CTAs where kThreads is the CTA
    const int side = (int)(item & 1);
    long long rest = item >> 1;
    const int h = (int)(rest % a.Hkv);
    rest /= a.Hkv;
    const int local = (int)(rest % a.items_per_seq);
    const int b = (int)(rest / a.items_per_seq);

    const int L = a.lens[b];
    const int t0 = a.cu ? a.cu[b] : b;
    const long long n = a.cu ? (long long)a.cu[b + 1] - t0 : 1;
    if (n == 0 || (!a.cu && L <= 0)) return;  // nothing new, or a padding entry of a step
    if (t0 < 0 || n < 0 || t0 + n > a.total || n > a.max_seqlen || L < n || L > ((long long)a.max_blocks << a.log2P)) {
        if (tid == 0 && local == 0) report_invalid();
        return;
    }
    const int start = L - (int)n;
    const int bi = (start >> a.log2P) + local;
    if (bi > (L - 1) >> a.log2P) return;
    const int block = a.table[(size_t)b * a.max_blocks + bi];
    if (block < 0 || block >= a.n_blocks) {
        if (tid == 0) report_invalid();
        return;
    }
    const int lo = max(start, bi << a.log2P);
    const int count = min(L, (bi + 1) << a.log2P) - lo;
    const int before = lo - (bi << a.log2P);  // tokens that the block holds already
    const int D8 = a.log2D - 3;
    const int vecs = count << D8;

    const T* x = static_cast<const T*>(a.x[side]) + (size_t)(t0 + (lo - start)) * a.stride_t[side] +
                 (size_t)h * a.stride_h[side];
    const size_t bh = (size_t)block * a.Hkv + h;
    uint8_t* codes = a.cache[side] + ((bh << a.log2P) << a.log2D);
    float* scale = a.scale[side] + bh;
    const float old = before > 0 ? *scale : 0.f;

    Raw8<T> raw[kAppendVecs];
    float amax = 0.f;
#pragma unroll
    for (int v = 0; v < kAppendVecs; ++v) {
        const int i = v * kThreads + tid;
        if (i < vecs) raw[v].load(x + (size_t)(i >> D8) * a.stride_t[side] + ((i & ((1 << D8) - 1)) << 3));
    }
#pragma unroll
    for (int v = 0; v < kAppendVecs; ++v) {
        if (v * kThreads + tid < vecs) {
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float m = fabsf(raw[v].get(u));
                amax = m <= 3.402823466e38f ? fmaxf(amax, m) : amax;  // infinities and NaN set no scale
            }
        }
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, m));
    if constexpr (kThreads > 32) {
        __shared__ float part[kThreads / 32];
        if ((tid & 31) == 0) part[tid >> 5] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) amax = fmaxf(amax, part[w]);
    }
    const float fits = kv8_scale_for(amax);
    const float s = fmaxf(old, fits);
    if (before > 0 && s > old) {
        const float ratio = old / s;
        uint4* c = reinterpret_cast<uint4*>(codes);
        for (int i = tid; i < before << (a.log2D - 4); i += kThreads) {
            uint4 w = c[i];
            uint32_t* e = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                uint32_t p0, p1;
                kv8_decode4(e[u], p0, p1);
                const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&p0));
                const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&p1));
                e[u] = kv8_encode2(f0.x * ratio, f0.y * ratio) | (kv8_encode2(f1.x * ratio, f1.y * ratio) << 16);
            }
            c[i] = w;
        }
    }
    if (tid == 0 && s != old) *scale = s;
    const float inv = 1.f / s;  // exact: a power of two
    uint8_t* dst = codes + ((size_t)before << a.log2D);
#pragma unroll
    for (int v = 0; v < kAppendVecs; ++v) {
        const int i = v * kThreads + tid;
        if (i < vecs) {
            uint2 w;
            w.x = kv8_encode2(raw[v].get(0) * inv, raw[v].get(1) * inv) |
                  (kv8_encode2(raw[v].get(2) * inv, raw[v].get(3) * inv) << 16);
            w.y = kv8_encode2(raw[v].get(4) * inv, raw[v].get(5) * inv) |
                  (kv8_encode2(raw[v].get(6) * inv, raw[v].get(7) * inv) << 16);
            *reinterpret_cast<uint2*>(dst + ((size_t)i << 3)) = w;
        }
    }
}

struct ReadArgs {
    const uint8_t* cache[2];
    const float* scale[2];
    const int* table;
    const int* cu;
    void* out[2];
    int max_seqlen, total, B, max_blocks, n_blocks, log2P, Hkv, log2D, blocks_per_seq;
    int chunks;  // CTAs for the codes of a block, K's or V's
};

constexpr int kReadThreads = 256;
constexpr int kReadVecs = 8;  // vectors a thread has in flight

// Codes -> values, 16 bytes of output a thread and vector.  A block's codes of all heads are one run
// of memory, and so are its tokens' values; a CTA takes kReadThreads * kReadVecs vectors of such a
// run, K's or V's, so that the chain of offsets, block id and codes is walked once for 16 KB of codes
// and every thread has all its loads under way before the first store.
template <typename T>
__global__ void __launch_bounds__(kReadThreads) kv8_read_kernel(const ReadArgs a) {
    constexpr int kVec = 16 / sizeof(T), kLog2Vec = sizeof(T) == 4 ? 2 : 3;
    grid_dependency_wait();
    allow_dependent_launch();
    unsigned rest = blockIdx.x;
    const int side = rest & 1;
    rest >>= 1;
    const int chunk = rest % (unsigned)a.chunks;
    rest /= (unsigned)a.chunks;
    const int bi = rest % (unsigned)a.blocks_per_seq, b = rest / (unsigned)a.blocks_per_seq;
    const int t0 = a.cu[b];
    const long long n = (long long)a.cu[b + 1] - t0;
    if (t0 < 0 || n < 0 || t0 + n > a.total || n > a.max_seqlen || n > ((long long)a.max_blocks << a.log2P)) {
        if (threadIdx.x == 0 && bi == 0) report_invalid();
        return;
    }
    const long long left = n - ((long long)bi << a.log2P);  // tokens from the block's first on
    if (left <= 0) return;
    const int block = a.table[(size_t)b * a.max_blocks + bi];
    if (block < 0 || block >= a.n_blocks) {
        if (threadIdx.x == 0) report_invalid();
        return;
    }
    const int log2_head = a.log2P + a.log2D;
    const uint8_t* src = (side ? a.cache[1] : a.cache[0]) + (((size_t)block * a.Hkv) << log2_head);
    const float* scales = (side ? a.scale[1] : a.scale[0]) + (size_t)block * a.Hkv;
    T* dst = static_cast<T*>(side ? a.out[1] : a.out[0]) + ((((size_t)t0 + ((size_t)bi << a.log2P)) * a.Hkv) << a.log2D);
    const int first = (chunk * (kReadVecs * kReadThreads) + threadIdx.x) << kLog2Vec;  // code in the run
    const int end = a.Hkv << log2_head;
    uint2 codes[kReadVecs];
    float scale[kReadVecs];
#pragma unroll
    for (int v = 0; v < kReadVecs; ++v) {
        const int i = first + ((v * kReadThreads) << kLog2Vec);
        if (i < end && ((i & ((1 << log2_head) - 1)) >> a.log2D) < left) {
            if constexpr (kVec == 8) {
                codes[v] = *reinterpret_cast<const uint2*>(src + i);
            } else {
                codes[v].x = *reinterpret_cast<const uint32_t*>(src + i);
            }
            scale[v] = scales[i >> log2_head];
        }
    }
#pragma unroll
    for (int v = 0; v < kReadVecs; ++v) {
        const int i = first + ((v * kReadThreads) << kLog2Vec);
        const int row = (i & ((1 << log2_head) - 1)) >> a.log2D;
        if (i >= end || row >= left) continue;
        float x[kVec];
#pragma unroll
        for (int u = 0; u < kVec / 4; ++u) {
            uint32_t p0, p1;
            kv8_decode4(u == 0 ? codes[v].x : codes[v].y, p0, p1);
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&p0));
            const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&p1));
            x[4 * u] = f0.x * scale[v];
            x[4 * u + 1] = f0.y * scale[v];
            x[4 * u + 2] = f1.x * scale[v];
            x[4 * u + 3] = f1.y * scale[v];
        }
        uint4 o;
        if constexpr (kVec == 8) {
            o.x = Elem<T>::pack2(x[0], x[1]);
            o.y = Elem<T>::pack2(x[2], x[3]);
            o.z = Elem<T>::pack2(x[4], x[5]);
            o.w = Elem<T>::pack2(x[6], x[7]);
        } else {
            o = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
        }
        T* to = dst + ((((size_t)row * a.Hkv) + (i >> log2_head)) << a.log2D) + (i & ((1 << a.log2D) - 1));
        *reinterpret_cast<uint4*>(to) = o;
    }
}

template <typename T>
int launch_append(const AppendArgs& a, long long values, cudaStream_t st) {
    // values: the most one item can hold.  A warp an item up to 2048 of them, else the CTA that
    // holds them at 64 a thread.
    const long long warp_grid = (a.items + 3) / 4;
    if (values <= 32 * 8 * kAppendVecs) return kv8_launch(kv8_append_kernel<T, 32>, dim3((unsigned)warp_grid), 128, 0, st, a);
    if (values <= 128 * 8 * kAppendVecs)
        return kv8_launch(kv8_append_kernel<T, 128>, dim3((unsigned)a.items), 128, 0, st, a);
    if (values <= 256 * 8 * kAppendVecs)
        return kv8_launch(kv8_append_kernel<T, 256>, dim3((unsigned)a.items), 256, 0, st, a);
    return kv8_launch(kv8_append_kernel<T, 512>, dim3((unsigned)a.items), 512, 0, st, a);
}

int ilog2(int x) {
    int r = 0;
    while ((1 << r) < x) ++r;
    return r;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace b200

B200_DEFINE_ERR_TAKER(kv8_cache, b200::g_err_kv8_cache)

extern "C" int kv8_append_sm100(const void* k, long long k_stride_token, long long k_stride_head, const void* v,
                                long long v_stride_token, long long v_stride_head, void* k_cache, void* v_cache,
                                float* k_scale, float* v_scale, const int* block_table, const int* seq_lens,
                                const int* cu_seqlens, int max_seqlen, int total_tokens, int B, int max_blocks,
                                int n_blocks, int block_size, int Hkv, int D, int in_dtype, void* stream) {
    using namespace b200;
    if (!k || !v || !seq_lens) return B200LAB_ERR_INVALID;
    int rc = kv8_check_cache(k_cache, v_cache, k_scale, v_scale, block_table, B, max_blocks, n_blocks, block_size, Hkv, D);
    if (rc != B200LAB_OK) return rc;
    if (in_dtype < B200LAB_F16 || in_dtype > B200LAB_F32) return B200LAB_ERR_INVALID;
    if (max_seqlen < 1 || total_tokens < 1) return B200LAB_ERR_INVALID;
    if (!cu_seqlens && (max_seqlen != 1 || total_tokens != B)) return B200LAB_ERR_INVALID;
    const int unit = in_dtype == B200LAB_F32 ? 4 : 8;  // values in 16 bytes
    if (!aligned16(k) || !aligned16(v) || k_stride_token % unit || k_stride_head % unit || v_stride_token % unit ||
        v_stride_head % unit || k_stride_token < 0 || k_stride_head < 0 || v_stride_token < 0 || v_stride_head < 0)
        return B200LAB_ERR_INVALID;
    AppendArgs a;
    a.x[0] = k, a.x[1] = v;
    a.stride_t[0] = k_stride_token, a.stride_t[1] = v_stride_token;
    a.stride_h[0] = k_stride_head, a.stride_h[1] = v_stride_head;
    a.cache[0] = static_cast<uint8_t*>(k_cache), a.cache[1] = static_cast<uint8_t*>(v_cache);
    a.scale[0] = k_scale, a.scale[1] = v_scale;
    a.table = block_table, a.lens = seq_lens, a.cu = cu_seqlens;
    const int most = max_seqlen < total_tokens ? max_seqlen : total_tokens;
    a.max_seqlen = most, a.total = total_tokens, a.B = B, a.max_blocks = max_blocks, a.n_blocks = n_blocks;
    a.log2P = kv8_log2_block(block_size), a.Hkv = Hkv, a.log2D = ilog2(D);
    const long long touched = ((long long)most + block_size - 2) / block_size + 1;  // `most` tokens from any slot on
    a.items_per_seq = (int)(touched < max_blocks ? touched : max_blocks);
    a.items = 2LL * B * a.items_per_seq * Hkv;
    if (a.items > 0x7fffffffLL) return B200LAB_ERR_UNSUPPORTED;
    rc = kv8_device().status;
    if (rc != B200LAB_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long long values = (long long)(most < block_size ? most : block_size) * D;
    switch (in_dtype) {
        case B200LAB_F16: return launch_append<__half>(a, values, st);
        case B200LAB_BF16: return launch_append<__nv_bfloat16>(a, values, st);
        default: return launch_append<float>(a, values, st);
    }
}

extern "C" int kv8_read_sm100(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                              const int* block_table, const int* cu_seqlens, int max_seqlen, int total_tokens, void* k,
                              void* v, int B, int max_blocks, int n_blocks, int block_size, int Hkv, int D,
                              int out_dtype, void* stream) {
    using namespace b200;
    if (!k || !v || !cu_seqlens) return B200LAB_ERR_INVALID;
    int rc = kv8_check_cache(k_cache, v_cache, k_scale, v_scale, block_table, B, max_blocks, n_blocks, block_size, Hkv, D);
    if (rc != B200LAB_OK) return rc;
    if (out_dtype < B200LAB_F16 || out_dtype > B200LAB_F32) return B200LAB_ERR_INVALID;
    if (max_seqlen < 1 || total_tokens < 1 || !aligned16(k) || !aligned16(v)) return B200LAB_ERR_INVALID;
    ReadArgs a;
    a.cache[0] = static_cast<const uint8_t*>(k_cache), a.cache[1] = static_cast<const uint8_t*>(v_cache);
    a.scale[0] = k_scale, a.scale[1] = v_scale;
    a.table = block_table, a.cu = cu_seqlens;
    a.out[0] = k, a.out[1] = v;
    const int most = max_seqlen < total_tokens ? max_seqlen : total_tokens;
    a.max_seqlen = most, a.total = total_tokens, a.B = B, a.max_blocks = max_blocks, a.n_blocks = n_blocks;
    a.log2P = kv8_log2_block(block_size), a.Hkv = Hkv, a.log2D = ilog2(D);
    const long long blocks = ((long long)most + block_size - 1) / block_size;
    a.blocks_per_seq = (int)(blocks < max_blocks ? blocks : max_blocks);
    const long long run = ((long long)Hkv * block_size * D) >> (out_dtype == B200LAB_F32 ? 2 : 3);  // vectors
    if (run > 0x10000000LL) return B200LAB_ERR_UNSUPPORTED;
    const long long per_cta = (long long)kReadThreads * kReadVecs;
    a.chunks = (int)((run + per_cta - 1) / per_cta);
    const long long grid = 2LL * B * a.blocks_per_seq * a.chunks;
    if (grid > 0x7fffffffLL) return B200LAB_ERR_UNSUPPORTED;
    rc = kv8_device().status;
    if (rc != B200LAB_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 g((unsigned)grid);
    switch (out_dtype) {
        case B200LAB_F16: return kv8_launch(kv8_read_kernel<__half>, g, kReadThreads, 0, st, a);
        case B200LAB_BF16: return kv8_launch(kv8_read_kernel<__nv_bfloat16>, g, kReadThreads, 0, st, a);
        default: return kv8_launch(kv8_read_kernel<float>, g, kReadThreads, 0, st, a);
    }
}
