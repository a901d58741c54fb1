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
    __device__ __forceinline__ void zero() { a = make_uint4(0, 0, 0, 0); }
    // The largest magnitude of some vectors' finite values.  Magnitudes of one sign order as their
    // bits do, so two values are compared at a time; only where an infinity or NaN turns up are the
    // values looked at one by one.
    template <int N> static __device__ __forceinline__ float amax(const Raw8 (&v)[N]) {
        constexpr uint32_t kInf = sizeof(T) == 2 && Elem<T>::kFmt == 0 ? 0x7c00u : 0x7f80u;
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            m = __vimax3_u16x2(m, v[i].a.x & 0x7fff7fffu, v[i].a.y & 0x7fff7fffu);
            m = __vimax3_u16x2(m, v[i].a.z & 0x7fff7fffu, v[i].a.w & 0x7fff7fffu);
        }
        uint32_t one = max(m & 0xffffu, m >> 16);
        if (one >= kInf) {
            one = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint16_t* e = reinterpret_cast<const uint16_t*>(&v[i].a);
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const uint32_t x = e[u] & 0x7fffu;
                    one = x < kInf ? max(one, x) : one;
                }
            }
        }
        const uint16_t bits = (uint16_t)one;
        return Elem<T>::to_f(*reinterpret_cast<const T*>(&bits));
    }
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
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    template <int N> static __device__ __forceinline__ float amax(const Raw8 (&v)[N]) {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float m = fabsf(v[i].get(u));
                most = m <= 3.402823466e38f ? fmaxf(most, m) : most;  // infinities and NaN set no scale
            }
        return most;
    }
};

// Division of n < 2^31 by a number the host knows: (n + umulhi(n, mul)) >> shift, with
// 2^shift >= d and mul = floor(2^32 (2^shift - d) / d) + 1.
struct Divisor {
    uint32_t d, mul, shift;
};
Divisor make_divisor(uint32_t d) {
    Divisor v = {d, 0, 0};
    while ((1ull << v.shift) < d) ++v.shift;
    v.mul = (uint32_t)((((1ull << v.shift) - d) << 32) / d + 1);
    return v;
}
__device__ __forceinline__ uint32_t divide(uint32_t& n, const Divisor& v) {  // leaves the remainder
    const uint32_t q = (n + __umulhi(n, v.mul)) >> v.shift, r = n - q * v.d;
    n = r;
    return q;
}

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
    Divisor by_head, by_local;
};

constexpr int kAppendVecs = 8;  // vectors of 8 values a thread holds: 32 registers of 16-bit values, 64 of fp32
constexpr int append_cta(int threads) { return threads < 128 ? 128 : threads; }
// CTAs an SM: 1024 threads of 64 registers, or 512 of 128
template <typename T> constexpr int append_resident(int threads) { return (sizeof(T) == 2 ? 1024 : 512) / append_cta(threads); }

// What one item of the writer is: `count` new tokens from x on, into the slots from `before` on of one
// head of a block, of K or V.
struct AppendItem {
    int side, h, token, count, before;
    int bh;  // block * Hkv + head
};
__device__ __forceinline__ AppendItem append_item(const AppendArgs& a, long long item) {
    AppendItem it = {0, 0, 0, 0, 0, 0};
    if (item >= a.items) return it;
    unsigned rest = (unsigned)item;
    it.side = rest & 1;
    rest >>= 1;
    uint32_t local = divide(rest, a.by_head);
    it.h = (int)rest;
    const int b = (int)divide(local, a.by_local);
    const int L = a.lens[b];
    const int t0 = a.cu ? a.cu[b] : b;
    const long long n = a.cu ? (long long)a.cu[b + 1] - t0 : 1;
    if (n == 0 || (!a.cu && L == 0)) return it;  // nothing new, or a padding entry of a step
    if (t0 < 0 || n < 0 || t0 + n > a.total || n > a.max_seqlen || L < n || L > ((long long)a.max_blocks << a.log2P)) {
        if (local == 0) report_invalid();
        return it;
    }
    const int start = L - (int)n;
    const int bi = (start >> a.log2P) + (int)local;
    if (bi > (L - 1) >> a.log2P) return it;
    const int block = a.table[(size_t)b * a.max_blocks + bi];
    if (block < 0 || block >= a.n_blocks) {
        report_invalid();
        return it;
    }
    const int lo = max(start, bi << a.log2P);
    it.token = t0 + (lo - start);
    it.count = (int)(min((long long)L, ((long long)bi + 1) << a.log2P) - lo);
    it.before = lo - (bi << a.log2P);
    it.bh = block * a.Hkv + it.h;
    return it;
}

// kThreads threads hold an item's values in registers (each is read once from memory), reduce their
// largest magnitude to the block's scale and write the codes.  A block begun by an earlier call keeps
// a larger old scale; where the new tokens need a larger one, its codes are rounded to it first.  Only
// slots below the sequence's length are written.
// Bound by memory for prompts, by latency for a step of one token a sequence, where a warp has an item.
// A grid of resident CTAs walks the items; each lane looks up one of the next 32 (a chain of two loads
// and a hundred instructions, which with an item a CTA were half of all that ran: 25k tokens of
// 8 sequences, D 128, 35 us so, 27 us now, 88 % of the bytes' time; 64k tokens of fp32, 8 heads of 128 or 4 of 256,
// 102 to 104 us, the measured copy rate), and items with nothing to write cost no more than that.
template <typename T, int kThreads>
__global__ void __launch_bounds__(append_cta(kThreads), append_resident<T>(kThreads))
    kv8_append_kernel(const AppendArgs a) {
    constexpr int kItems = kThreads < 128 ? 128 / kThreads : 1;  // of a CTA at a time
    __shared__ float part[2][kThreads / 32];
    grid_dependency_wait();
    allow_dependent_launch();
    const int tid = threadIdx.x % kThreads, lane = threadIdx.x & 31;
    const int log2_row = a.log2D - 3;  // vectors of a row
    const long long stride = (long long)gridDim.x * kItems;
    int turn = 0;
    for (long long item = (long long)blockIdx.x * kItems + threadIdx.x / kThreads; item < a.items; item += 32 * stride) {
        const AppendItem mine = append_item(a, item + lane * stride);
        for (unsigned some = __ballot_sync(0xffffffffu, mine.count > 0); some; some &= some - 1, turn ^= 1) {
            // the same item for all its threads: every warp of it has looked up the same ones
            const int from = __ffs(some) - 1;
            const int side = __shfl_sync(0xffffffffu, mine.side, from), h = __shfl_sync(0xffffffffu, mine.h, from);
            const int count = __shfl_sync(0xffffffffu, mine.count, from);
            const int before = __shfl_sync(0xffffffffu, mine.before, from);
            const size_t token = __shfl_sync(0xffffffffu, mine.token, from), bh = __shfl_sync(0xffffffffu, mine.bh, from);
            const long long stride_t = side ? a.stride_t[1] : a.stride_t[0];
            // this thread's vectors: one every kThreads >> log2_row rows, in the same channels
            const int row = tid >> log2_row, rows = kThreads >> log2_row;
            const T* x = static_cast<const T*>(side ? a.x[1] : a.x[0]) + (token + row) * stride_t +
                         (size_t)h * (side ? a.stride_h[1] : a.stride_h[0]) + ((tid & ((1 << log2_row) - 1)) << 3);
            uint8_t* codes = (side ? a.cache[1] : a.cache[0]) + ((bh << a.log2P) << a.log2D);
            float* scale = (side ? a.scale[1] : a.scale[0]) + bh;
            Raw8<T> raw[kAppendVecs];
            const float old = before > 0 ? *scale : 0.f;
#pragma unroll
            for (int v = 0; v < kAppendVecs; ++v) {
                raw[v].zero();
                if (row + v * rows < count) raw[v].load(x + v * (rows * stride_t));
            }
            float amax = Raw8<T>::amax(raw);
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, m));
            if constexpr (kThreads > 32) {
                // two sets in turn: what is read here is written again only after the next item's barrier
                if ((tid & 31) == 0) part[turn][tid >> 5] = amax;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kThreads / 32; ++w) amax = fmaxf(amax, part[turn][w]);
            }
            const float s = fmaxf(old, kv8_scale_for(amax));
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
                        e[u] = kv8_encode4(f0.x * ratio, f0.y * ratio, f1.x * ratio, f1.y * ratio);
                    }
                    c[i] = w;
                }
            }
            if constexpr (kThreads == 32) __syncwarp();  // every lane has read the old scale
            if (tid == 0 && s != old) *scale = s;
            const float inv = 1.f / s;  // exact: a power of two
            uint8_t* dst = codes + ((size_t)before << a.log2D) + tid * 8;
#pragma unroll
            for (int v = 0; v < kAppendVecs; ++v) {
                if (row + v * rows < count) {
                    uint2 w;
                    w.x = kv8_encode4(raw[v].get(0) * inv, raw[v].get(1) * inv, raw[v].get(2) * inv, raw[v].get(3) * inv);
                    w.y = kv8_encode4(raw[v].get(4) * inv, raw[v].get(5) * inv, raw[v].get(6) * inv, raw[v].get(7) * inv);
                    *reinterpret_cast<uint2*>(dst + v * (kThreads * 8)) = w;
                }
            }
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

// Codes -> values, 16 bytes of output a thread and vector.  Bound by memory: 87k tokens, D 128, to bf16 in
// 87 us (6.2 TB/s, 96 % of the measured copy rate; 202 us with the items' chain walked by every thread
// for four vectors); 64k tokens of 8 heads of 128 to fp32 in 106 us (98 %).  A block's codes of all heads are one run
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

template <typename T, int kThreads> int launch_append_as(const AppendArgs& a, int sms, cudaStream_t st) {
    constexpr int kCta = append_cta(kThreads), kItems = kCta / kThreads;
    // as many CTAs as are resident, each with about the same number of items
    const long long ctas = (a.items + kItems - 1) / kItems, most = (long long)sms * append_resident<T>(kThreads);
    return kv8_launch(kv8_append_kernel<T, kThreads>, dim3((unsigned)(ctas < most ? ctas : most)), kCta, 0, st, a);
}

template <typename T> int launch_append(const AppendArgs& a, long long values, int sms, cudaStream_t st) {
    // values: the most one item can hold.  A warp an item up to 2048 of them, else the CTA that
    // holds them at 64 a thread.
    constexpr int kEach = 8 * kAppendVecs;
    if (values <= 32 * kEach) return launch_append_as<T, 32>(a, sms, st);
    if (values <= 128 * kEach) return launch_append_as<T, 128>(a, sms, st);
    if (values <= 256 * kEach) return launch_append_as<T, 256>(a, sms, st);
    return launch_append_as<T, 512>(a, sms, st);
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
    a.by_head = make_divisor((uint32_t)Hkv);
    a.by_local = make_divisor((uint32_t)a.items_per_seq);
    const Kv8Device dev = kv8_device();
    rc = dev.status;
    if (rc != B200LAB_OK) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long long values = (long long)(most < block_size ? most : block_size) * D;
    switch (in_dtype) {
        case B200LAB_F16: return launch_append<__half>(a, values, dev.sms, st);
        case B200LAB_BF16: return launch_append<__nv_bfloat16>(a, values, dev.sms, st);
        default: return launch_append<float>(a, values, dev.sms, st);
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
    if (run > 0x8000000LL) return B200LAB_ERR_UNSUPPORTED;  // a code's place in the run fits 31 bits
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
