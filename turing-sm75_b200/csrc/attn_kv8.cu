// attn_kv8.cu -- softmax attention of a batch's last tokens over the paged 8-bit key/value cache
// (layout and number format: kv8.cuh).
//
// No counterpart in the reference, which attends over dense 16-bit K and V
// (src/attn_sm75.cu:107-112); same softmax semantics as attn_fwd_sm100.
//
// Mathematics.  For a query row r and key j, with the codes c and the scales sK, sV of j's block:
//   x = scale log2(e) sK (q . cK) + log2(sV),  p = 2^(x - m),  O = sum p cV,  l = sum p / sV,
// m a reference of the row's, and o = O / l.  The scale of V rides in the exponent of the weights,
// so codes are multiplied as they are, whatever the blocks' scales.
// The products take p in fp16, which has 40 powers of two where a long row's weights, times scales of
// 2^-40 to 2^40, span any number.  So m is no running maximum: it follows the keys in hand, up and down.
// p stays below 2^15, and the largest p of a piece (the 16 or 32 keys a warp takes at a time) above 2^-8, so that
// a rounding to fp16 is off by 2^-11 of the weight or 2^-17 of its piece's largest, however small the piece's
// weights are beside the row's others: many small weights together count in full.  m goes no lower than where
// l, in fp32, would pass 2^60; what fp16 loses of a weight there moves an output by less than 448 x 2^-83.
// (With a running maximum for m, a warp that met a key 2^26 above its others lost all of those.  What following the
// keys costs: 0.5 % of long streams, 3 to 6 % of short calls, 7 % of many rows at D 256.)
//
// What bounds it: the bytes of the cache; a code is used by the few rows of its kv group only
// (2 x rows flop a byte).  Everything follows from streaming them:
//   * The batch's work is cut into equal runs of key tiles, one run a CTA, whatever the lengths are
//     (the tiles of all (sequence, kv-head, row tile) segments are numbered through on the device, and
//     a segment counts two or three tiles more than it has, for its start and end: ragged B64 108 us without,
//     99 with).  A segment that lies in one run is written out by its CTA; one that is cut leaves fp32
//     partial sums in the workspace, two at most a CTA, and a second kernel joins them.
//   * Where there are few short segments, the chain of plan, parts and second kernel is most of a call: there
//     a cluster of CTAs has a segment, and joins its sums through distributed shared memory.
//   * A warp has a ring of its own of 16- or 32-key pieces of K and V, which its lanes fill with
//     16-byte asynchronous copies, whose next pieces are requested across segment borders, so that
//     the loads never pause.  Nothing but the joins holds the warps of a CTA together.  (TMA boxes
//     into the same rings measured the same on the largest batches and slower on short rings of
//     small boxes: four drafted tokens x 16 sequences of 2-4k 35.0 against 33.7 us.)
//   * Products are mma.sync m16n8k16 with the KEYS (S^T = K Q^T) and the CHANNELS (O^T = V^T P^T)
//     on the 16-row side and 8 query rows on the 8-column side: a kv group of 1..8 rows fills one
//     column tile, a code is converted to fp16 (exactly) once for all column tiles, and P^T
//     turns from result into operand by a register transpose (movmatrix).
//   * The channel and key order inside a product is free: each thread takes 32 consecutive channels
//     of a K row (two 16-byte shared loads, conflict-free as the chunks are swizzled) and 16 of four V
//     rows, whose bytes it pairs by key with one PRMT for two conversions.
//   * No lane asks the others for a row's largest score while each finds its own in the range of m.
//   * Q is brought to fp16 with a power of two a row: exact, as bf16 and fp16 both have at most 11
//     significant bits (below 2^-29 of the row's largest value, bits are lost).
// Measured, 32 q-heads on 8 kv-heads of 128 unless said, calls back to back in a graph: B64 x 16k 345 us
// (6.2 TB/s, 97 % of the measured copy rate), B64 x 400..8k 99.6 us (88 %), B1 x 16k 14.6 us, B1 x 1000
// 6.2 us, 4 tokens x B16 x 2-4k 32 us, 24 q-heads on 4 of 256 with gate B32 x 2-4k 43 us, 8 heads of 64
// B48 x 250..2500 23 us.  The longest streams are bound by memory; what the shorter ones add to that is
// a call's own chain (lengths, block ids, codes; the part's join; the second kernel: 7 us in all, 4 with clusters).
// With more rows or 64 channels it is latency: a piece is a chain of dependent conversions, products and
// exponentials, and the two or four warps that a scheduler has cover a third or a half of it (issue 34 and 48 %
// busy, half of the stalls waits for a fixed latency; neither a pipe nor memory is full).
#include "errwords.h"
#include "kv8.cuh"

namespace b200 {
namespace {

__device__ int g_err_attn_kv8 = 0;

constexpr int kMostWarps = 4;             // of a CTA that goes by the plan
constexpr int kWideWarps = 8;             // of a wide CTA of a cluster
constexpr int kMostCluster = 8;           // CTAs of a cluster
constexpr int kGroup = 16;                // keys of one product
constexpr float kLog2e = 1.4426950408889634f;
// A row's reference m is moved when a score lies above m + kTop, to kRise below it, or when a piece has none as high
// as m + kBottom, to kFall above its largest: whole powers of two away, so that fp16 holds the weight of the key that moved
// it as it is.  (References that are whole numbers themselves, moved without a rounding, leave the largest weights rounded
// where l is not: errors of fp16 outputs 3.0e-4 instead of 2.2e-4, and a lone key's values no longer exact.)
constexpr float kTop = 15.f, kRise = 10.f, kBottom = -8.f, kFall = 4.f;
constexpr int kMostSum = 60;              // and not to where its sum l would pass 2^60

// What a variant's CTA works on and holds; `ctas` (of four warps) fill an SM's registers and shared
// memory.  Two groups a piece halve what a piece costs beside its products where registers allow it
// (one column tile of D 128: B64 x 16k 424 us with one group and two CTAs, 348 with two and three; two
// column tiles: 41 us with one and three CTAs, 35 with two and two; D 256: 46 us with one, 59 with two).
struct Shape {
    int groups;  // of a piece, the keys a warp takes at a time
    int ctas;
    int depth;   // pieces of a warp's ring
};
constexpr Shape shape_of(int D, int nt) {
    return D == 64 ? (nt == 1 ? Shape{2, 4, 2} : Shape{2, 3, 3}) : D == 128 ? (nt == 1 ? Shape{2, 3, 2} : Shape{2, 2, 2}) : Shape{1, 2, 2};
}
template <int D, int NT, int W> struct Cfg {  // W: warps of a CTA
    static constexpr int kH = shape_of(D, NT).groups;
    static constexpr int kPiece = kGroup * kH;
    static constexpr int kTile = kPiece * W;                // keys a CTA takes at a time
    static constexpr int kBytes = 2 * kPiece * D;           // a piece of K, then one of V
    static constexpr int kCtas = shape_of(D, NT).ctas * kMostWarps / W;
    static constexpr int kDepth = shape_of(D, NT).depth;
    // channels joined at a time: as many as leave room for the CTAs (D 256: 42.8 us with 128, 43.0 with 64)
    static constexpr int kRow = D == 256 || (D == 128 && NT == 2) ? 128 : 64;
    // what a segment's start and end cost, in tiles (a tile of D 256 has a group a warp, and its sums are
    // the longest to join: 45.4 us with 2 and a ring of three, 43.0 with 3 and a ring of two)
    static constexpr int kStart = D == 256 ? 3 : 2;
};

struct alignas(16) GroupMeta {  // of 16 keys
    float ks, vs;   // scales of K and V
    int ok;         // 0: no key of the group is in the sequence, or its block id lies outside the pool
    int unused;
};

struct Args {
    const void* q;
    const void* g;  // gate or null
    void* o;
    long long q_st, q_sh, g_st, g_sh;  // strides of a token and of a head
    int g_aligned;  // the gate's rows lie on 16 bytes
    const uint8_t* k;
    const uint8_t* v;
    const int* table;
    const int* lens;
    const int* cu;  // null: one query token a sequence
    const float* k_scale;
    const float* v_scale;
    float* part;    // [grid][2][rows][D] sums, [grid][2][rows] (m, l)
    int* meta;      // [grid][4]: what a CTA says of its last segment (end of attn_kv8_kernel)
    int rts;        // row tiles that a sequence can have
    int log2C;      // CTAs of a cluster that has a segment; negative: the segments are cut by a plan
    int max_seqlen_q, total_q, B, max_blocks, n_blocks, log2P, Hq, Hkv, group, causal;
    uint32_t head_bytes;  // of a block's codes of one head: block_size * D
    float scale;
};

// ---- the plan: sequences -> segments -> key tiles ----------------------------------------------
struct Seq {
    int n, L, t0;      // query tokens, keys, first packed token
    int tiles, rts;    // key tiles and row tiles
    // in the numbering of the plan, where a segment counts kStart tiles more than it has
    template <int kStart> __device__ __forceinline__ long long units(int Hkv) const {
        return tiles ? (long long)(tiles + kStart) * rts * Hkv : 0;
    }
};

// A sequence whose offsets or length are outside what the call was given has no tiles and is reported.
template <int D, int NT, int W> __device__ __forceinline__ Seq load_seq(const Args& a, int b, bool report) {
    Seq s;
    s.L = a.lens[b];
    s.t0 = a.cu ? a.cu[b] : b;
    const long long n = a.cu ? (long long)a.cu[b + 1] - s.t0 : 1;
    s.tiles = s.rts = s.n = 0;
    if (n == 0) return s;
    if (s.t0 < 0 || n < 0 || s.t0 + n > a.total_q || n > a.max_seqlen_q || s.L < 0 ||
        s.L > ((long long)a.max_blocks << a.log2P)) {
        if (report) atomicExch(&g_err_attn_kv8, B200LAB_ERR_INVALID);
        return s;
    }
    s.n = (int)n;
    constexpr int kTile = Cfg<D, NT, W>::kTile;
    s.tiles = max(1, (s.L + kTile - 1) / kTile);  // a sequence without keys has a tile, to write its zeros
    s.rts = (s.n * a.group + 8 * NT - 1) / (8 * NT);
    return s;
}

// A place in the numbered tiles: sequence, kv-head, row tile, key tile (negative: in the kStart units
// that stand for the segment's start); `left` units of the CTA's run from here on.
template <int D, int NT, int W> struct Cursor {
    Seq s;
    int b, h, rt, tile, left;  // (a CTA's run fits 32 bits: 2^31 tiles would take it hours)
    // the CTA's tiles of this segment: [first, first + count), none where count <= 0
    __device__ __forceinline__ int span() const { return min(s.tiles - tile, left); }
    __device__ __forceinline__ int first() const { return max(tile, 0); }
    __device__ __forceinline__ int count() const { return tile + span() - first(); }
    // to the next segment
    __device__ __forceinline__ void next(const Args& a) {
        left -= span();
        if (left <= 0) return;
        tile = -Cfg<D, NT, W>::kStart;
        if (++rt < s.rts) return;
        rt = 0;
        if (++h < a.Hkv) return;
        h = 0;
        do {
            s = load_seq<D, NT, W>(a, ++b, false);
        } while (s.tiles == 0);  // ends: tiles are left
    }
};

// Sums of the lanes up to and including this one.
__device__ __forceinline__ long long scan(long long x, int lane) {
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const long long other = __shfl_up_sync(0xffffffffu, x, m);
        if (lane >= m) x += other;
    }
    return x;
}

// The units [0, total) dealt to G CTAs: total % G CTAs have one more than the others.
struct Deal {
    long long each, more;
    Deal() = default;
    __device__ __forceinline__ Deal(long long total, int G) {
        // 32-bit division, a fraction of the 64-bit one's time, wherever it does
        each = total <= 0x7fffffffLL ? (long long)((uint32_t)total / (uint32_t)G) : total / G;
        more = total - each * G;
    }
    __device__ __forceinline__ long long start(int c) const { return c * each + min((long long)c, more); }
    __device__ __forceinline__ int holder(long long unit) const {
        const long long big = more * (each + 1);  // units of the CTAs that have one more
        if (unit < big) return (int)(unit / (each + 1));
        return (int)(more + (unit - big) / each);
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <int D, int NT, int W> struct Smem {
    using C = Cfg<D, NT, W>;
    alignas(128) uint8_t ring[W][C::kDepth][C::kBytes];
    alignas(16) float join[W > 1 ? W : 1][W > 1 ? 8 : 1][W > 1 ? C::kRow + 4 : 4];
    uint2 qfrag[NT > 1 ? NT : 1][NT > 1 ? D / 16 : 1][32];
    GroupMeta meta[W][C::kDepth][C::kH];
    float m[W][8 * NT], l[W][8 * NT];
    float qscale[8 * NT];
};

// The factor that brings a part's sums from its own level m to the largest one M.  A part without scores counts
// nothing, one whose scores are all NaN (l is NaN) everything.  Every part has an l of 1 to 2 times the parts that it
// is made of: what underflows counts less than 2^-126 of the sum.
__device__ __forceinline__ float part_weight(float m, float l, float M) {
    return m == -INFINITY && l == l ? 0.f : ex2(m - M);
}

// Row n of a row tile -> query token of the sequence and head of the group.
__device__ __forceinline__ void row_place(int row, int group, int& i, int& hg) {
    i = row / group;
    hg = row - i * group;
}

// kPer consecutive channels of a row: the gate's, and the gated outputs' store.
template <typename T, int kPer> struct Channels {
    alignas(sizeof(T) * kPer) T v[kPer];
    __device__ __forceinline__ void load_gate(const Args& a, size_t token, int head, int d0) {
        const T* g = static_cast<const T*>(a.g) + token * a.g_st + (size_t)head * a.g_sh + d0;
        if (a.g_aligned) {  // d0 is a multiple of kPer
            if constexpr (kPer == 8) {
                *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(g);
            } else if constexpr (kPer == 4) {
                *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(g);
            } else {
                *reinterpret_cast<uint32_t*>(v) = *reinterpret_cast<const uint32_t*>(g);
            }
        } else {
#pragma unroll
            for (int u = 0; u < kPer; ++u) v[u] = g[u];
        }
    }
};
// Stores channels of a row whose sums are x and `sum`.  A row that sees no key (sum 0) is 0 whatever its gate: a padding
// entry's may be NaN.
template <typename T, int kPer>
__device__ __forceinline__ void store_row(const Args& a, size_t token, int head, int D, int d0, const float (&x)[kPer],
                                          float sum, const Channels<T, kPer>& gate) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    float y[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
        y[u] = x[u] * inv;
        if (a.g && sum != 0.f) y[u] = y[u] / (1.f + __expf(-Elem<T>::to_f(gate.v[u])));
    }
    uint32_t w[kPer / 2];
#pragma unroll
    for (int u = 0; u < kPer; u += 2) w[u / 2] = Elem<T>::pack2(y[u], y[u + 1]);
    uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<T*>(a.o) + (token * a.Hq + head) * (size_t)D + d0);
    if constexpr (kPer == 8) {
        *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
    } else if constexpr (kPer == 4) {
        *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
    } else {
        static_assert(kPer == 2, "");
        *o = w[0];
    }
}

// Where a 16-byte chunk of a row lies in a piece: chunk index XOR row (XOR half the row at D = 64,
// where two rows share a line of banks).
template <int D> __device__ __forceinline__ int chunk_at(int row, int chunk) {
    if constexpr (D == 64) {
        return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
    } else {
        return row * 128 + ((chunk ^ (row & 7)) << 4);
    }
}

// The key that row i (mod 8) of a product stands for.  At D = 64, where a row is half a line of
// banks, this order keeps the K loads (rows i and i + 1 of the product) and the V loads (rows 0, 2,
// 4, 6, or 1, 3, 5, 7) free of bank conflicts; wider rows need none.
template <int D> __device__ __forceinline__ int key_of(int i) {
    return D == 64 ? (int)((0x65742130u >> (4 * i)) & 7u) : i;
}

// One query row's channels of this thread, as the operand of Q K^T: f[ks] holds the channels that
// word ks of the thread's K row holds.  The row is scaled by a power of two to a largest magnitude
// in [2^14, 2^15); returned is the inverse factor, NaN for a row that is not finite (its scores then
// are NaN, as in exact arithmetic some would be).  q null: a row of zeros.
template <int D, typename T>
__device__ __forceinline__ float load_q(const T* q, int t, uint32_t (&f)[D / 16][2]) {
    constexpr int kBoxes = D > 128 ? 2 : 1, kDims = D == 64 ? 16 : 32;  // channels a thread has in a box
    uint4 raw[kBoxes][kDims / 8];
    float amax = 0.f;
    bool finite = true;
#pragma unroll
    for (int box = 0; box < kBoxes; ++box)
#pragma unroll
        for (int c = 0; c < kDims / 8; ++c) {
            raw[box][c] = q ? *reinterpret_cast<const uint4*>(q + box * 128 + t * kDims + c * 8) : make_uint4(0, 0, 0, 0);
            const T* e = reinterpret_cast<const T*>(&raw[box][c]);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float x = fabsf(Elem<T>::to_f(e[u]));
                finite = finite && x <= 3.402823466e38f;
                amax = fmaxf(amax, x);
            }
        }
#pragma unroll
    for (int m = 1; m <= 2; m <<= 1) {  // the four threads of a row
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, m));
        finite = __shfl_xor_sync(0xffffffffu, (int)finite, m) && finite;
    }
    const uint32_t field = min(268u - min(__float_as_uint(amax) >> 23, 254u), 227u);
    const float to = finite ? __uint_as_float(field << 23) : 0.f;
#pragma unroll
    for (int box = 0; box < kBoxes; ++box)
#pragma unroll
        for (int c = 0; c < kDims / 8; ++c) {
            const T* e = reinterpret_cast<const T*>(&raw[box][c]);
            float x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = finite ? Elem<T>::to_f(e[u]) * to : 0.f;
            const int ks = box * (kDims / 4) + 2 * c;
            f[ks][0] = pack_h2(x[0], x[1]);
            f[ks][1] = pack_h2(x[2], x[3]);
            f[ks + 1][0] = pack_h2(x[4], x[5]);
            f[ks + 1][1] = pack_h2(x[6], x[7]);
        }
    return finite ? __uint_as_float((254u - field) << 23) : __uint_as_float(0x7fc00000u);
}

// 16 or 4 bytes global -> shared without waiting.
__device__ __forceinline__ void copy16(uint32_t smem, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(void* smem, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending> __device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// Barrier of a cluster's threads: what they wrote to shared memory before is read by all after it.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address in CTA `rank` of the cluster of what lies at `smem` in this one, and loads from there.
__device__ __forceinline__ uint32_t cluster_at(uint32_t smem, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t at) {
    float2 x;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(at) : "memory");
    return x;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t at) {
    float4 x;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
    return x;
}

// The pieces of one warp in the order it takes them, requested ahead of their use.
template <int D, int NT, int W> struct Producer {
    using C = Cfg<D, NT, W>;
    Cursor<D, NT, W> c;
    int k;        // next tile of the segment, from c.first()
    int block;    // lane i: block * Hkv + head of group i of the next 32 / kH pieces; -1: none
    uint32_t to;  // where this lane's first 16 bytes of a group go in a piece

    // Requests the next piece, if one is left, into a ring slot, as one group of copies.
    __device__ __forceinline__ void issue(const Args& a, uint8_t* slot, GroupMeta* meta, int warp, int lane) {
        while (c.left > 0 && !(k < c.count() && (c.first() + k) * C::kTile + warp * C::kPiece < c.s.L)) {
            c.next(a);
            k = 0;
        }
        if (c.left > 0) {
            constexpr int kAhead = 32 / C::kH;
            if ((k & (kAhead - 1)) == 0) {  // the blocks of the next pieces, a group a lane
                const int pos = (c.first() + k + lane / C::kH) * C::kTile + warp * C::kPiece + (lane % C::kH) * kGroup;
                block = -1;
                if (k + lane / C::kH < c.count() && pos < c.s.L) {
                    block = a.table[(size_t)c.b * a.max_blocks + (pos >> a.log2P)];
                    if (block < 0 || block >= a.n_blocks) {
                        atomicExch(&g_err_attn_kv8, B200LAB_ERR_INVALID);
                        block = -1;
                    } else {
                        block = block * a.Hkv + c.h;
                    }
                }
            }
            const int first = (k & (kAhead - 1)) * C::kH;  // lane of the piece's first group
            if (lane >= first && lane < first + C::kH) {
                GroupMeta* m = meta + (lane - first);
                m->ok = block >= 0;
                // a scale is stored or copied, never both: nothing orders a store before an asynchronous
                // copy of the same thread to the same address
                if (block >= 0) {
                    copy4(&m->ks, a.k_scale + block);
                    copy4(&m->vs, a.v_scale + block);
                } else {
                    m->ks = m->vs = 1.f;
                }
            }
            const uint32_t dst = smem_u32(slot);
#pragma unroll
            for (int u = 0; u < C::kH; ++u) {
                const int bh = __shfl_sync(0xffffffffu, block, first + u);
                if (bh < 0) continue;
                const int row = ((c.first() + k) * C::kTile + warp * C::kPiece + u * kGroup) & ((1 << a.log2P) - 1);
                const size_t at = (size_t)(uint32_t)bh * a.head_bytes + (uint32_t)(row * D + lane * 16);
                const uint8_t *from_k = a.k + at, *from_v = a.v + at;
#pragma unroll
                for (int i = 0; i < kGroup * D / 512; ++i) {  // 512 contiguous bytes a copy of the warp: 512 / D rows
                    constexpr int kBox = D > 128 ? 128 : D, kStep = 512 / D;
                    // rows i * kStep further: the same place in a row, chunk index XOR what the row adds to it
                    constexpr uint32_t kTurn = D == 64 ? 0u : (uint32_t)(kStep & 7) << 4;
                    const uint32_t off = (to ^ ((i * kTurn) & 0x70u)) + (uint32_t)((u * kGroup + i * kStep) * kBox);
                    copy16(dst + off, from_k + i * 512);
                    copy16(dst + C::kPiece * D + off, from_v + i * 512);
                }
            }
            ++k;
        }
        copy_commit();
    }
};

// The codes of V of a group that some row does not see whole, before their product.  Behind the
// sequence's last key lies whatever was there: its codes count as 0, as 0 * NaN is NaN.  A NaN that
// some rows see must not reach the rows that do not: it is taken out of the product, and the sums of
// the rows that see it become NaN here.
//   w: this thread's codes of the keys r[0..3] of the group; row: row g of the first column tile
template <int D, int NT, int kBoxes, int kWords>
__device__ __forceinline__ void take_out_masked(const Args& a, const Seq& s, uint32_t (&w)[kBoxes][4][kWords],
                                                float (&o)[NT][D / 16][4], const int (&r)[4], int base, bool ok, int row) {
    uint32_t nan = 0;
#pragma unroll
    for (int box = 0; box < kBoxes; ++box)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                if (base + r[q] >= s.L || !ok) w[box][q][j] = 0;
                nan |= ((w[box][q][j] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
            }
    if (__builtin_expect(!__any_sync(0xffffffffu, nan != 0), 1)) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int sees = min(a.causal ? s.L - s.n + (row + nt * 8) / a.group + 1 : s.L, s.L);
        uint32_t vis[2];
#pragma unroll
        for (int q = 0; q < 2; ++q)
            vis[q] = pack_h2(base + r[2 * q] < sees ? 1.f : 0.f, base + r[2 * q + 1] < sees ? 1.f : 0.f);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const int box = i / (2 * kWords), j = (i % (2 * kWords)) >> 1;
            uint32_t f[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t at = ((w[box][q][j] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                f[q] = (at >> 7) * 0x38u;  // 1.0 where a NaN is
            }
            const uint32_t sel = (i & 1) ? 0x7362u : 0x5140u;
            const uint32_t x = __byte_perm(f[0], f[1], sel), y = __byte_perm(f[2], f[3], sel);
            float hit[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t a0, a1, a2, a3;
            kv8_decode4(x, a0, a1);
            kv8_decode4(y, a2, a3);
            mma(hit, a0, a1, a2, a3, vis[0], vis[1]);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (hit[c] > 0.f) o[nt][i][c] = __uint_as_float(0x7fc00000u);
        }
    }
#pragma unroll
    for (int box = 0; box < kBoxes; ++box)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                const uint32_t at = ((w[box][q][j] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                w[box][q][j] &= ~((at >> 7) * 0xffu);
            }
}

// kCluster: a cluster has a segment, its CTAs equal runs of the segment's tiles; they read one another's
// sums and write the outputs, so that there is no plan and no second kernel.
template <int D, int NT, int W, bool kCluster, typename T>
__global__ void __launch_bounds__(32 * W, Cfg<D, NT, W>::kCtas)
    attn_kv8_kernel(const Args a) {
    using C = Cfg<D, NT, W>;
    constexpr int kRows = 8 * NT, kDepth = C::kDepth, kH = C::kH, kPiece = C::kPiece, kTile = C::kTile;
    constexpr int kBox = D > 128 ? 128 : D, kBoxes = D / kBox;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    Smem<D, NT, W>& sm = *reinterpret_cast<Smem<D, NT, W>*>(smem_raw);
    const int tid = threadIdx.x, warp = W > 1 ? tid >> 5 : 0, lane = tid & 31;
    const int g = lane >> 2, t = lane & 3;

    // Launched early, but lets the join kernel start only as its CTAs end (the default): a join CTA that
    // waits on an SM keeps the next call's CTA from starting there (B64 16k, calls back to back: 580 us
    // with the trigger here, 350 without).
    grid_dependency_wait();

    // ---- this CTA's run of tiles.  Every warp finds it for itself: a lane adds up the sequences of its
    // share, then the share that holds the run's first unit is looked at, a sequence a lane
    Cursor<D, NT, W> cur;
    Deal deal;
    long long u1 = 0;
    const int rank = kCluster ? blockIdx.x & ((1 << a.log2C) - 1) : 0;
    if constexpr (kCluster) {
        const int segment = blockIdx.x >> a.log2C, bh = segment / a.rts;
        cur.rt = segment - bh * a.rts;
        cur.b = bh / a.Hkv;
        cur.h = bh - cur.b * a.Hkv;
        cur.s = load_seq<D, NT, W>(a, cur.b, cur.h == 0 && cur.rt == 0);
        if (cur.rt >= cur.s.rts) return;  // the whole cluster
        cur.tile = (int)((long long)cur.s.tiles * rank >> a.log2C);
        cur.left = (int)((long long)cur.s.tiles * (rank + 1) >> a.log2C) - cur.tile;
    } else {
        const int share = (a.B + 31) / 32;
        Seq s = {0, 0, 0, 0, 0};
        long long mine = 0;
    #pragma unroll 4
        for (int b = min(a.B, lane * share), i = 0; i < share && b < a.B; ++i, ++b) {
            s = load_seq<D, NT, W>(a, b, blockIdx.x == 0);
            mine += s.template units<C::kStart>(a.Hkv);
        }
        long long upto = scan(mine, lane);
        const long long total = __shfl_sync(0xffffffffu, upto, 31);
        const int G = (int)min((long long)gridDim.x, total);
        if ((int)blockIdx.x >= G) {
            if (tid == 0) a.meta[4 * blockIdx.x] = -1;
            return;
        }
        deal = Deal(total, G);
        const long long u0 = deal.start(blockIdx.x);
        u1 = deal.start(blockIdx.x + 1);
        int from = __ffs(__ballot_sync(0xffffffffu, u0 < upto)) - 1;  // there is one: u0 < total
        cur.b = from * share;
        long long before = __shfl_sync(0xffffffffu, upto - mine, from);  // units before the sequence in hand
        if (share > 1) {
            const int end = min(a.B, cur.b + share);
            for (int b = cur.b + lane;; b += 32) {
                s.tiles = 0;
                if (b < end) s = load_seq<D, NT, W>(a, b, false);
                mine = s.template units<C::kStart>(a.Hkv);
                upto = scan(mine, lane);
                const unsigned past = __ballot_sync(0xffffffffu, u0 < before + upto);
                if (past) {  // ends: the share holds u0
                    from = __ffs(past) - 1;
                    cur.b = __shfl_sync(0xffffffffu, b, from);
                    before += __shfl_sync(0xffffffffu, upto - mine, from);
                    break;
                }
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        cur.s.n = __shfl_sync(0xffffffffu, s.n, from);
        cur.s.L = __shfl_sync(0xffffffffu, s.L, from);
        cur.s.t0 = __shfl_sync(0xffffffffu, s.t0, from);
        cur.s.tiles = __shfl_sync(0xffffffffu, s.tiles, from);
        cur.s.rts = __shfl_sync(0xffffffffu, s.rts, from);
        {
            // the segment and the tile in it; a sequence's units fit 32 bits nearly always
            const long long local = u0 - before;
            const int per = cur.s.tiles + C::kStart;
            const long long seg = local <= 0x7fffffffLL ? (long long)((uint32_t)local / (uint32_t)per) : local / per;
            cur.tile = (int)(local - seg * per) - C::kStart;
            cur.h = (int)(seg / cur.s.rts);
            cur.rt = (int)(seg - (long long)cur.h * cur.s.rts);
            cur.left = (int)(u1 - u0);
        }
    }

    Producer<D, NT, W> pro;
    pro.c = cur;
    pro.k = 0;
    {
        constexpr int kRowLanes = D / 16, kBoxLanes = kBox / 16;
        const int chunk = lane % kRowLanes;
        pro.to = (chunk / kBoxLanes) * (kPiece * kBox) + chunk_at<D>(lane / kRowLanes, chunk % kBoxLanes);
    }
    // where this thread's codes lie in a group: chunks of K's rows key(g) (key(g) + 8: 8 rows further), of
    // V's rows key(2t) and key(2t + 1)
    const int kr = key_of<D>(g);
    const int k_at = chunk_at<D>(kr, D == 64 ? t : 2 * t);
    const int v_at[2] = {D == 64 ? chunk_at<D>(key_of<D>(2 * t), g >> 1) + (g & 1) * 8 : chunk_at<D>(2 * t, g),
                         D == 64 ? chunk_at<D>(key_of<D>(2 * t + 1), g >> 1) + (g & 1) * 8 : chunk_at<D>(2 * t + 1, g)};
    int slot = 0;  // the next piece's
    for (int i = 0; i < kDepth; ++i) pro.issue(a, sm.ring[warp][i], sm.meta[warp][i], warp, lane);

    int said = -1;  // whether the run's last segment goes on in the next CTA's, and where it begins
    for (bool once = kCluster; once || cur.left > 0; once = false, cur.next(a)) {
        const int first = cur.first(), run = cur.count();
        if (!kCluster && run <= 0) continue;  // the cut lies in the segment's start: the next CTA has it
        const Seq& s = cur.s;
        const int row0 = cur.rt * kRows, rows = min(kRows, s.n * a.group - row0);

        // ---- Q
        uint32_t qf[NT == 1 ? D / 16 : 1][2];
        float qs[NT][2];  // score factors of this thread's two columns of each column tile
        {
            const float to_log2 = a.scale * kLog2e;
            if constexpr (NT == 1) {
                const T* q = nullptr;
                if (g < rows) {
                    int i, hg;
                    row_place(row0 + g, a.group, i, hg);
                    q = static_cast<const T*>(a.q) + (size_t)(s.t0 + i) * a.q_st + (size_t)(cur.h * a.group + hg) * a.q_sh;
                }
                const float f = load_q<D, T>(q, t, qf) * to_log2;
                qs[0][0] = __shfl_sync(0xffffffffu, f, 8 * t);
                qs[0][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
            } else {
                for (int nt = warp; nt < NT; nt += W) {
                    const T* q = nullptr;
                    if (nt * 8 + g < rows) {
                        int i, hg;
                        row_place(row0 + nt * 8 + g, a.group, i, hg);
                        q = static_cast<const T*>(a.q) + (size_t)(s.t0 + i) * a.q_st +
                            (size_t)(cur.h * a.group + hg) * a.q_sh;
                    }
                    uint32_t f[D / 16][2];
                    const float x = load_q<D, T>(q, t, f) * to_log2;
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) sm.qfrag[nt][ks][lane] = make_uint2(f[ks][0], f[ks][1]);
                    if (t == 0) sm.qscale[nt * 8 + g] = x;
                }
                __syncthreads();  // written again only after the join below, which ends with one too
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    qs[nt][0] = sm.qscale[nt * 8 + 2 * t];
                    qs[nt][1] = sm.qscale[nt * 8 + 2 * t + 1];
                }
            }
        }
        float m[NT][2], l[NT][2], o[NT][D / 16][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        }
        // the first key that some row of this row tile does not see
        const int all_see = a.causal ? s.L - s.n + row0 / a.group + 1 : s.L;

        for (int k = 0; k < run; ++k) {
            const int base = (first + k) * kTile + warp * kPiece;
            if (base >= s.L) break;
            copy_wait<kDepth - 1>();
            __syncwarp();
            {
                const uint8_t* ks_ = sm.ring[warp][slot];
                const uint8_t* vs_ = ks_ + kPiece * D;
                // scale of K, log2 and inverse of the scale of V: powers of two, whose exponents are read off
                // (a scale that is none takes the long way)
                float gk[kH], gl[kH], gi[kH];
                bool ok[kH], whole_piece = true;
#pragma unroll
                for (int u = 0; u < kH; ++u) {
                    const GroupMeta m = sm.meta[warp][slot][u];
                    const float v = fminf(fmaxf(m.vs, kKv8MinScale), kKv8MaxScale);
                    const uint32_t bits = __float_as_uint(v);
                    gk[u] = m.ks;
                    gl[u] = (float)((int)(bits >> 23) - 127);
                    gi[u] = __uint_as_float((254u << 23) - bits);
                    if (__builtin_expect(bits & 0x7fffffu, 0)) gl[u] = log2f(v), gi[u] = 1.f / v;
                    ok[u] = m.ok;
                    whole_piece = whole_piece && m.ok;
                }
                // ---- S^T = K Q^T (16 keys x 8 rows a group and column tile); a lone group has two partial
                // sums, to shorten the chain of products
                constexpr int kAcc = kH == 1 ? 2 : 1;
                float sc[kH][NT][kAcc][4];
#pragma unroll
                for (int u = 0; u < kH; ++u)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            sc[u][nt][0][i] = 0.f;
                            sc[u][nt][kAcc - 1][i] = 0.f;
                        }
#pragma unroll
                for (int box = 0; box < kBoxes; ++box) {
                    constexpr int kChunks = D == 64 ? 1 : 2;
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
                        for (int u = 0; u < kH; ++u) {
                            const uint8_t* kb = ks_ + (box * kPiece + u * kGroup) * kBox;
                            // the other chunk of the pair is the swizzled index with its last bit turned
                            const uint4 lo = *reinterpret_cast<const uint4*>(kb + (k_at ^ (c * 16)));
                            const uint4 hi = *reinterpret_cast<const uint4*>(kb + (k_at ^ (c * 16)) + 8 * kBox);
                            const uint32_t w0[4] = {lo.x, lo.y, lo.z, lo.w}, w1[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int ks = (box * kChunks + c) * 4 + j;
                                uint32_t a0, a1, a2, a3;
                                kv8_decode4(w0[j], a0, a2);
                                kv8_decode4(w1[j], a1, a3);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    if constexpr (NT == 1) {
                                        mma(sc[u][nt][ks & (kAcc - 1)], a0, a1, a2, a3, qf[ks][0], qf[ks][1]);
                                    } else {
                                        const uint2 qb = sm.qfrag[nt][ks][lane];
                                        mma(sc[u][nt][ks & (kAcc - 1)], a0, a1, a2, a3, qb.x, qb.y);
                                    }
                                }
                            }
                        }
                    }
                }
                // ---- softmax over the piece: thread (g, t) has keys key(g), key(g) + 8 of each group and rows
                // 2t, 2t + 1
                const bool edge = base + kPiece > all_see || !whole_piece;  // some key is masked for some row
                bool out = false;  // this thread's largest score of some row is not in the range of the row's m
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int u = 0; u < kH; ++u) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = kAcc == 2 ? sc[u][nt][0][i] + sc[u][nt][kAcc - 1][i] : sc[u][nt][0][i];
                            sc[u][nt][0][i] = fmaf(x, qs[nt][i & 1] * gk[u], gl[u]);
                        }
                        if (__builtin_expect(edge, 0)) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int key = base + u * kGroup + kr + (i >> 1) * 8;
                                const int row = row0 + nt * 8 + 2 * t + (i & 1);
                                const int sees = a.causal ? s.L - s.n + row / a.group + 1 : s.L;
                                if (key >= min(sees, s.L) || !ok[u]) sc[u][nt][0][i] = -INFINITY;
                            }
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float x = fmaxf(sc[0][nt][0][c], sc[0][nt][0][c + 2]);
#pragma unroll
                        for (int u = 1; u < kH; ++u) x = fmaxf(x, fmaxf(sc[u][nt][0][c], sc[u][nt][0][c + 2]));
                        out |= !(fabsf(x - m[nt][c] - (kTop + kBottom) / 2) <= (kTop - kBottom) / 2);
                    }
                }
                if (__builtin_expect(__any_sync(0xffffffffu, out), 0)) {
                    float x[NT][2], to[NT][2];  // of each row: the largest score of all lanes, and the new m
                    bool fall = false;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            x[nt][c] = fmaxf(sc[0][nt][0][c], sc[0][nt][0][c + 2]);
#pragma unroll
                            for (int u = 1; u < kH; ++u) x[nt][c] = fmaxf(x[nt][c], fmaxf(sc[u][nt][0][c], sc[u][nt][0][c + 2]));
#pragma unroll
                            for (int k = 4; k <= 16; k <<= 1) x[nt][c] = fmaxf(x[nt][c], __shfl_xor_sync(0xffffffffu, x[nt][c], k));
                            to[nt][c] = x[nt][c] > m[nt][c] + kTop ? x[nt][c] - kRise : m[nt][c];
                            fall |= x[nt][c] > -INFINITY && x[nt][c] < m[nt][c] + kBottom;
                        }
                    if (__any_sync(0xffffffffu, fall)) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                float sum = l[nt][c];
#pragma unroll
                                for (int k = 4; k <= 16; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
                                // (a sum that is NaN has the largest exponent: m stays)
                                const int room = kMostSum - 1 - ((int)(__float_as_uint(sum) >> 23) - 127);
                                if (x[nt][c] > -INFINITY && x[nt][c] < m[nt][c] + kBottom)
                                    to[nt][c] = fmaxf(x[nt][c] + kFall, m[nt][c] - (float)max(room, 0));
                            }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (!__any_sync(0xffffffffu, to[nt][0] != m[nt][0] || to[nt][1] != m[nt][1])) continue;
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float f = to[nt][c] == m[nt][c] ? 1.f : ex2(m[nt][c] - to[nt][c]);
                            m[nt][c] = to[nt][c];
                            l[nt][c] *= f;
#pragma unroll
                            for (int i = 0; i < D / 16; ++i) {
                                o[nt][i][c] *= f;
                                o[nt][i][c + 2] *= f;
                            }
                        }
                    }
                }
                uint32_t pb[kH][NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0];
                    const float m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
                    for (int u = 0; u < kH; ++u) {
                        const float p0 = ex2(sc[u][nt][0][0] - m0), p1 = ex2(sc[u][nt][0][1] - m1);
                        const float p2 = ex2(sc[u][nt][0][2] - m0), p3 = ex2(sc[u][nt][0][3] - m1);
                        l[nt][0] = fmaf(p0 + p2, gi[u], l[nt][0]);
                        l[nt][1] = fmaf(p1 + p3, gi[u], l[nt][1]);
                        // the weights are rounded to fp16, of which the head of this file says how much it costs; the
                        // sum l takes them before
                        pb[u][nt][0] = transpose8x8(pack_h2(p0, p1));
                        pb[u][nt][1] = transpose8x8(pack_h2(p2, p3));
                    }
                }
                // ---- O^T += V^T P^T: product rows are channels, k index i stands for key key(i)
                const int r[4] = {key_of<D>(2 * t), key_of<D>(2 * t + 1), key_of<D>(2 * t) + 8, key_of<D>(2 * t + 1) + 8};
                constexpr int kWords = kBox / 32;  // of a thread in a V row
#pragma unroll
                for (int u = 0; u < kH; ++u) {
                    uint32_t w[kBoxes][4][kWords];
#pragma unroll
                    for (int box = 0; box < kBoxes; ++box)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            // rows key(2t), key(2t + 1), and those 8 further, which are swizzled alike
                            const uint8_t* vb = vs_ + (box * kPiece + u * kGroup + (q >> 1) * 8) * kBox + v_at[q & 1];
                            if constexpr (D == 64) {
                                const uint2 x = *reinterpret_cast<const uint2*>(vb);
                                w[box][q][0] = x.x, w[box][q][1] = x.y;
                            } else {
                                const uint4 x = *reinterpret_cast<const uint4*>(vb);
                                w[box][q][0] = x.x, w[box][q][1] = x.y, w[box][q][2] = x.z, w[box][q][3] = x.w;
                            }
                        }
                    if (__builtin_expect(edge, 0)) take_out_masked<D, NT>(a, s, w, o, r, base + u * kGroup, ok[u], row0 + g);
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        const int box = i / (kBox / 16), j = (i % (kBox / 16)) >> 1;
                        const uint32_t sel = (i & 1) ? 0x7362u : 0x5140u;
                        const uint32_t x = __byte_perm(w[box][0][j], w[box][1][j], sel);
                        const uint32_t y = __byte_perm(w[box][2][j], w[box][3][j], sel);
                        uint32_t a0, a1, a2, a3;
                        kv8_decode4(x, a0, a1);
                        kv8_decode4(y, a2, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma(o[nt][i], a0, a1, a2, a3, pb[u][nt][0], pb[u][nt][1]);
                    }
                }
                __syncwarp();  // every lane has read the slot
                pro.issue(a, sm.ring[warp][slot], sm.meta[warp][slot], warp, lane);
            }
            if (++slot == kDepth) slot = 0;
        }

        // ---- the sums of this run's part of the segment
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int x = 4; x <= 16; x <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], x);
        const bool whole = first == 0 && run == s.tiles;
        if (W > 1 || !whole) {
            // to be joined: m lies anywhere below the weights that make l; here it becomes their level, by a power of two
            // that brings l to [1, 2) (no scores: l is 0 and m -infinity, and both stay)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t field = min(__float_as_uint(l[nt][c]) >> 23, 253u);
                    const float f = __uint_as_float((254u - field) << 23);
                    m[nt][c] += (float)((int)field - 127);
                    l[nt][c] *= f;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        o[nt][i][c] *= f;
                        o[nt][i][c + 2] *= f;
                    }
                }
        }
        constexpr int kOwn = kBox / 8;  // consecutive channels a thread has in a box, of rows 2t and 2t + 1
        if constexpr (kCluster) {
            // every warp leaves its sums in its own ring, from which nothing is read any more: a row's
            // channels, then its maximum and sum
            constexpr int kStride = D + 4;
            static_assert(kRows * kStride * 4 <= kDepth * C::kBytes, "");
            __syncwarp();
            float* own = reinterpret_cast<float*>(sm.ring[warp]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float* to = own + (nt * 8 + 2 * t + c) * kStride;
                    if (g == 0) *reinterpret_cast<float2*>(to + D) = make_float2(m[nt][c], l[nt][c]);
#pragma unroll
                    for (int e = 0; e < D / 32; ++e) {  // 4 channels at a time
                        const int box = e / (kOwn / 4), i = box * (kBox / 16) + (e % (kOwn / 4)) * 2;
                        *reinterpret_cast<float4*>(to + box * kBox + kOwn * g + (e % (kOwn / 4)) * 4) =
                            make_float4(o[nt][i][c], o[nt][i][c + 2], o[nt][i + 1][c], o[nt][i + 1][c + 2]);
                    }
                }
            cluster_sync();
            // as many threads as CTAs share four channels of a row, each with the sums of one CTA's warps (with two
            // shares under way a thread the tiles before them spill, 8 % slower).  A row is a multiple of 16 shares, so in
            // clusters of two and more, whose threads exchange values, a warp is in the loop as a whole
            constexpr int kVecs = D / 4, kThreads = 32 * W;
            const int from = tid & ((1 << a.log2C) - 1);
            const uint32_t theirs = cluster_at(smem_u32(sm.ring), from);
            for (int at = (rank * kThreads + tid) >> a.log2C; at < rows * kVecs; at += kThreads) {
                const int n = at / kVecs, d = (at % kVecs) * 4;
                int i, hg;
                row_place(row0 + n, a.group, i, hg);
                const size_t token = (size_t)(s.t0 + i);
                const int head = cur.h * a.group + hg;
                Channels<T, 4> gate;
                if (a.g && from == 0) gate.load_gate(a, token, head, d);
                float4 v[W];
                float2 ml[W];
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t row = theirs + w * (kDepth * C::kBytes) + n * (kStride * 4);
                    v[w] = cluster_load4(row + d * 4);
                    ml[w] = cluster_load2(row + D * 4);
                }
                float M = ml[0].x, sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 1; w < W; ++w) M = fmaxf(M, ml[w].x);
#pragma unroll
                for (int k = 1; k < kMostCluster; k <<= 1)
                    if (k < 1 << a.log2C) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float f = part_weight(ml[w].x, ml[w].y, M);
                    sum = fmaf(f, ml[w].y, sum);
                    x[0] = fmaf(f, v[w].x, x[0]);
                    x[1] = fmaf(f, v[w].y, x[1]);
                    x[2] = fmaf(f, v[w].z, x[2]);
                    x[3] = fmaf(f, v[w].w, x[3]);
                }
#pragma unroll
                for (int k = 1; k < kMostCluster; k <<= 1) {
                    if (k >= 1 << a.log2C) break;
                    sum += __shfl_xor_sync(0xffffffffu, sum, k);
#pragma unroll
                    for (int u = 0; u < 4; ++u) x[u] += __shfl_xor_sync(0xffffffffu, x[u], k);
                }
                if (from == 0) {
                    store_row<T, 4>(a, token, head, D, d, x, sum, gate);
                }
            }
            cluster_sync();  // the others have read this CTA's sums
            continue;
        }
        const int part = blockIdx.x * 2 + (first == 0 ? 1 : 0);
        float2* part_ml = reinterpret_cast<float2*>(a.part + (size_t)gridDim.x * 2 * kRows * D) + (size_t)part * kRows;
        if constexpr (W == 1) {
            // no other warp's to add: from the registers to where they belong
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int n = nt * 8 + 2 * t + c;
                    if (n >= rows) continue;
                    int i, hg;
                    row_place(row0 + n, a.group, i, hg);
                    const size_t token = (size_t)(s.t0 + i);
                    const int head = cur.h * a.group + hg;
                    if (!whole && g == 0) part_ml[n] = make_float2(m[nt][c], l[nt][c]);
#pragma unroll
                    for (int e = 0; e < D / 64; ++e) {  // 8 channels at a time
                        const int box = e / (kOwn / 8), from = (e % (kOwn / 8)) * 8, ch = box * kBox + kOwn * g + from;
                        float x[8];
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            x[2 * u] = o[nt][box * (kBox / 16) + from / 2 + u][c];
                            x[2 * u + 1] = o[nt][box * (kBox / 16) + from / 2 + u][c + 2];
                        }
                        if (whole) {
                            Channels<T, 8> gate;
                            if (a.g) gate.load_gate(a, token, head, ch);
                            store_row<T, 8>(a, token, head, D, ch, x, l[nt][c], gate);
                        } else {
                            float4* p = reinterpret_cast<float4*>(a.part + ((size_t)part * kRows + n) * D + ch);
                            p[0] = make_float4(x[0], x[1], x[2], x[3]);
                            p[1] = make_float4(x[4], x[5], x[6], x[7]);
                        }
                    }
                }
            __syncwarp();  // qfrag is read no more
        } else {
        // the other warps' are added by way of shared memory, kRow channels at a time
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c)
                if (g == 0) {
                    sm.m[warp][nt * 8 + 2 * t + c] = m[nt][c];
                    sm.l[warp][nt * 8 + 2 * t + c] = l[nt][c];
                }
        __syncthreads();
        constexpr int kRow = C::kRow, kPer = kRow / 16;
        const int jr = tid >> 4, jd = (tid & 15) * kPer;  // this thread's row of a column tile, and channels
        static_assert(W == 4 || kCluster, "8 rows x 16 threads");  // (clusters have gone on above)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float f[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int n = nt * 8 + 2 * t + c;
                float M = sm.m[0][n];
#pragma unroll
                for (int w = 1; w < W; ++w) M = fmaxf(M, sm.m[w][n]);
                f[c] = part_weight(m[nt][c], l[nt][c], M);
            }
#pragma unroll
            for (int d = 0; d < D / kRow; ++d) {
                constexpr int kSharers = kRow / kOwn, kJoins = kBox / kRow;
                if (g / kSharers == d % kJoins) {
#pragma unroll
                    for (int i = 0; i < kOwn / 2; i += 2) {
                        const float(&x)[4] = o[nt][(d / kJoins) * (kBox / 16) + i];
                        const float(&y)[4] = o[nt][(d / kJoins) * (kBox / 16) + i + 1];
                        *reinterpret_cast<float4*>(&sm.join[warp][2 * t][kOwn * (g % kSharers) + 2 * i]) =
                            make_float4(x[0] * f[0], x[2] * f[0], y[0] * f[0], y[2] * f[0]);
                        *reinterpret_cast<float4*>(&sm.join[warp][2 * t + 1][kOwn * (g % kSharers) + 2 * i]) =
                            make_float4(x[1] * f[1], x[3] * f[1], y[1] * f[1], y[3] * f[1]);
                    }
                }
                __syncthreads();
                const int n = nt * 8 + jr;
                if (n < rows) {
                    float M = sm.m[0][n];
#pragma unroll
                    for (int w = 1; w < W; ++w) M = fmaxf(M, sm.m[w][n]);
                    float sum = 0.f;
#pragma unroll
                    for (int w = 0; w < W; ++w)
                        sum += sm.l[w][n] * part_weight(sm.m[w][n], sm.l[w][n], M);
                    float x[kPer];
#pragma unroll
                    for (int u = 0; u < kPer; ++u) x[u] = 0.f;
#pragma unroll
                    for (int w = 0; w < W; ++w)
#pragma unroll
                        for (int u = 0; u < kPer; ++u) x[u] += sm.join[w][jr][jd + u];
                    if (whole) {
                        int i, hg;
                        row_place(row0 + n, a.group, i, hg);
                        const size_t token = (size_t)(s.t0 + i);
                        const int head = cur.h * a.group + hg;
                        Channels<T, kPer> gate;
                        if (a.g) gate.load_gate(a, token, head, d * kRow + jd);
                        store_row<T, kPer>(a, token, head, D, d * kRow + jd, x, sum, gate);
                    } else {
                        float* p = a.part + ((size_t)part * kRows + n) * D + d * kRow + jd;
#pragma unroll
                        for (int u = 0; u < kPer; u += 4)
                            *reinterpret_cast<float4*>(p + u) = make_float4(x[u], x[u + 1], x[u + 2], x[u + 3]);
                        if (d == 0 && jd == 0) part_ml[n] = make_float2(M, sum);
                    }
                }
                __syncthreads();
            }
        }
        }
        // A CTA that has the first tiles of a segment, and not the last, owns it and describes it: the CTA that has its
        // last tile, its place, its rows.  One with tiles of its middle alone names the owner, one without either says -1.
        if (tid == 0 && first + run < s.tiles) {
            const long long at = u1 - cur.left - cur.tile;  // tile 0 in the plan's numbering
            if (first == 0) {
                said = deal.holder(at + s.tiles - 1);
                a.meta[4 * blockIdx.x + 1] = s.t0;
                a.meta[4 * blockIdx.x + 2] = cur.h * a.group;
                a.meta[4 * blockIdx.x + 3] = row0 | rows << 24;
            } else {
                said = -2 - deal.holder(at);
            }
        }
    }
    if (!kCluster && tid == 0) a.meta[4 * blockIdx.x] = said;
}

// Joins the segments that were cut: part 0 of each is its owner's second one, the others are the first
// ones of the CTAs that follow, up to `last`.  Two forms, by how many segments there are:
//   many (kFew false): block (c, y), rows 8 y .. of the segment that CTA c owns, if it owns one; a warp a
//     row, as segments of like lengths have few parts (B4 x 8k, 4 tokens, eleven parts: 25.4 us so, 28.4 the other
//     way).  One far longer than the others has nearly all CTAs' parts: from kLong parts on, its rows go to the
//     blocks of its first CTAs, which own no segment, a row a block, whose warps share its parts (B64, one of
//     128k keys and 63 of 10, 4 heads on 1: 73 us with a warp a row, 23 so; B256, 128k and 255 of 500: 120, 101).
//   few: block (i, n), row n of the i-th segment that was cut, which the block looks up among the owners;
//     sixteen warps share the parts, of which there can be as many as CTAs.  (A block for every CTA and row
//     is a thousand blocks more to start: B1 x 64k, 16 heads on 1, 21.8 us with them, 17 without.)
// Either way a warp has the loads of kJoinAhead parts under way at once, behind the one of the segment's description.
constexpr int kJoinAhead = 4;
constexpr int kLong = 16;  // at least 8: the owner and seven that are neither it nor the last
template <int D, int NT, typename T, bool kFew>
__global__ void __launch_bounds__(kFew ? 512 : 256) attn_kv8_join_kernel(const Args a, int grid) {
    constexpr int kRows = 8 * NT, kVec = D / 32;  // channels of a lane
    constexpr int kWarps = kFew ? 16 : 8;
    grid_dependency_wait();
    allow_dependent_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int c = blockIdx.x;
    if constexpr (kFew) {
        __shared__ int owners[16], found;
        int before = 0, wanted = blockIdx.x;
        if (threadIdx.x == 0) found = -1;
        for (int i0 = 0; i0 < grid; i0 += 512) {
            const int i = i0 + threadIdx.x;
            const unsigned own = __ballot_sync(0xffffffffu, i < grid && a.meta[4 * i] >= 0);
            __syncthreads();  // the last chunk's owners are read
            if (lane == 0) owners[warp] = __popc(own);
            __syncthreads();
            int mine = before;
#pragma unroll
            for (int w = 0; w < 16; ++w) {
                if (w < warp) mine += owners[w];
                before += owners[w];
            }
            if ((own >> lane & 1) && mine + __popc(own & ((1u << lane) - 1)) == wanted) found = i;
        }
        __syncthreads();
        c = found;
        if (c < 0) return;
    }
    int4 desc = reinterpret_cast<const int4*>(a.meta)[c];
    int ahead_of = 0;  // which of the segment's CTAs this block stands for
    if (!kFew && desc.x < -1) {
        ahead_of = c + 2 + desc.x;
        if (ahead_of >= 8) return;
        c -= ahead_of;
        desc = reinterpret_cast<const int4*>(a.meta)[c];
    }
    const int last = desc.x, row0 = desc.w & 0xffffff, rows = desc.w >> 24;
    if (last < 0) return;
    const bool shared = kFew || last - c >= kLong;  // all warps have one row
    if (!shared && ahead_of > 0) return;
    const int n = kFew ? blockIdx.y : blockIdx.y * 8 + (shared ? ahead_of : warp);
    const int sharers = shared ? kWarps : 1, share = shared ? warp : 0;
    const int parts = n < rows ? last - c + 1 : 0;
    int i, hg;
    row_place(row0 + n, a.group, i, hg);
    const size_t token = (size_t)(desc.y + i);
    const int head = desc.z + hg;
    Channels<T, kVec> gate;
    if (a.g && n < rows) gate.load_gate(a, token, head, lane * kVec);
    const float2* ml = reinterpret_cast<const float2*>(a.part + (size_t)grid * 2 * kRows * D);
    float M = -INFINITY, sum = 0.f, x[kVec];
#pragma unroll
    for (int u = 0; u < kVec; ++u) x[u] = 0.f;
    for (int p0 = share; p0 < parts; p0 += sharers * kJoinAhead) {
        float2 st[kJoinAhead];
        float y[kJoinAhead][kVec];
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            const int p = min(p0 + j * sharers, parts - 1);  // past the end: the last one, not counted
            const size_t at = (size_t)(p == 0 ? 2 * c + 1 : 2 * (c + p)) * kRows + n;
            st[j] = ml[at];
            if (p0 + j * sharers >= parts) st[j] = make_float2(-INFINITY, 0.f);
            const float* src = a.part + at * D + lane * kVec;
#pragma unroll
            for (int u = 0; u < kVec; u += 2) {
                const float2 v = *reinterpret_cast<const float2*>(src + u);
                y[j][u] = v.x;
                y[j][u + 1] = v.y;
            }
        }
        float to = M;
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) to = fmaxf(to, st[j].x);
        const float f = part_weight(M, sum, to);
        sum *= f;
#pragma unroll
        for (int u = 0; u < kVec; ++u) x[u] *= f;
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            if (p0 + j * sharers >= parts) continue;
            const float w = part_weight(st[j].x, st[j].y, to);
            sum = fmaf(w, st[j].y, sum);
#pragma unroll
            for (int u = 0; u < kVec; ++u) x[u] = fmaf(w, y[j][u], x[u]);
        }
        M = to;
    }
    if (shared) {
        __shared__ float acc[kWarps][D];
        __shared__ float2 stat[kWarps];
        if (lane == 0) stat[warp] = make_float2(M, sum);
#pragma unroll
        for (int u = 0; u < kVec; ++u) acc[warp][lane * kVec + u] = x[u];
        __syncthreads();
        if (warp != 0) return;
        float all = M;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) all = fmaxf(all, stat[w].x);
        const float f = part_weight(M, sum, all);
        sum *= f;
#pragma unroll
        for (int u = 0; u < kVec; ++u) x[u] *= f;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            const float2 st = stat[w];
            const float g = part_weight(st.x, st.y, all);
            sum = fmaf(g, st.y, sum);
#pragma unroll
            for (int u = 0; u < kVec; ++u) x[u] = fmaf(g, acc[w][lane * kVec + u], x[u]);
        }
    }
    if (n >= rows) return;
    store_row<T, kVec>(a, token, head, D, lane * kVec, x, sum, gate);
}

// Column tiles of 8 query rows a CTA works on at once; rows beyond take further passes over the keys,
// which then come from L2.  Two tiles share the conversions but leave registers for fewer warps: they
// pay from 17 rows on (B32, 2-4k keys, D 128, 32 rows: 74 us with two, 81 with one, 95 with four, 16
// rows 34 with either), and never at D = 256 (16 rows: 51 us with one, 62 with two, which spill).
int column_tiles(int rows, int D) { return D == 256 || rows <= 8 ? 1 : 2; }

int plan_grid(int D, int nt, int warps, int sms) {
    return shape_of(D, nt).ctas * kMostWarps / warps * sms;
}

// Warps of a CTA.  Four share the tiles of a segment and join their sums in shared memory, which
// leaves few cut segments; a warp on its own joins nothing, and while it starts or ends a segment the
// SM's other warps go on: better where segments are short and many.  The lengths are on the device, so
// the rule goes by what the host has, the segments and the most that the block table can hold.  Measured
// by the plan, inputs in turn beyond L2, with four / with one, 32 q-heads on 8 kv-heads of 128 unless said: B64 x 200
// tokens 18.0 / 17.4 us, B128 x 200 27.0 / 23.6, B256 x 200 42.6 / 33.7, B512 x 64 51 / 30, B128 x 2k D 64 32 heads
// 190 / 177, and the other way B32 x 200 11.7 / 13.8.  A wide table does not tell what lengths it holds: B256 in one for
// 4k tokens is 42.6 / 33.7 where all have 200, 62.4 / 59.4 where they have 500, but 93 / 102 with 1000 and 180 / 192 with
// 200 to 4k.  The rule takes one there: up to 9 % lost where sequences are long, up to 21 % won where they are short.
int warps_of(long long segments, long long tokens, int D, int nt, int sms) {
    const long long alone = plan_grid(D, nt, 1, sms);
    return segments >= (tokens <= 512 ? alone / 2 : alone) ? 1 : 4;
}

// The clusters that work on a segment each: log2 of their CTAs, or -1 where the segments go by the plan, and a
// CTA's warps.  A cluster saves the plan and the second kernel, 2.5 to 4 us of a call's chain; the plan has all
// SMs on few segments and equal runs where lengths differ.  Which it is goes by the segments and by the most
// key tiles that one can have (by the block table: the lengths are on the device).  A cluster is as wide as gives
// an SM one CTA.  Where a CTA then has more than two tiles, eight warps share them, if the segments are so
// many that the clusters are pairs at most (wider ones of such CTAs do not all find room at once: B2 x 4096
// 16.4 us with eight CTAs of eight warps, 9.8 of four); else two CTAs an SM do, from four tiles on.
// Measured, 32 q-heads on 8 kv-heads of 128, planned / by clusters: B1 x 64 7.4 / 4.4 us, B1 x 1000 9.3 / 6.6,
// B1 x 4096 10.3 / 9.5, B1 x 8192 11.3 / 13.5 (so planned), B4 x 2000 12.5 / 9.5, B16 x 250 10.6 / 6.4, B32 x 250
// 11.6 / 7.0, B64 x 250 19.9 / 16.6, B128 x 200 23.5 / 23.0 (about even from here on: planned); with four warps /
// eight: B8 x 1000 9.2 / 8.3, B16 x 500 8.5 / 7.1, B1 x 2000 7.3 / 8.0 (so four).  Two column tiles: 4 tokens x B16 x 250
// planned 13.1, by clusters 8.7, x B16 x 1000 19.9 / 14.8, x B1 x 2000 11.1 / 12.8 (so planned).
struct Clusters {
    int log2C, warps;
};
Clusters clusters_of(long long segments, long long tokens, int D, int nt, int sms) {
    const Shape shape = shape_of(D, nt);
    const int tile = kGroup * shape.groups * kMostWarps, widest = nt == 1 ? 3 : 2, most = nt == 1 ? 4 : 2;
    const long long tiles = (tokens + tile - 1) / tile;
    if (segments > 4LL * sms || tiles > 8 * kMostCluster) return {-1, 0};
    int log2C = 0;
    while (log2C < widest && 1 << log2C < tiles && segments << (log2C + 1) <= sms) ++log2C;
    const long long wide = (long long)sms * (shape.ctas * kMostWarps / kWideWarps);  // places of eight warps
    if (log2C <= 1 && segments << log2C <= wide && tiles > 2LL << log2C && tiles <= 8LL << log2C)
        return {log2C, kWideWarps};
    if (log2C < widest && tiles > (long long)most << log2C && segments << (log2C + 1) <= 2LL * sms) ++log2C;
    if (tiles > (long long)most << log2C) return {-1, 0};
    return {log2C, kMostWarps};
}

// Lets a kernel have its shared memory, once a device.
template <typename Kern> int raise_smem(Kern kern, size_t smem, int device, std::atomic<unsigned long long>& ready) {
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (!bit || !(ready.load(std::memory_order_relaxed) & bit)) {
        B200_TRY_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    return B200LAB_OK;
}

size_t workspace_bytes(int D, int nt, int grid) {
    const size_t rows = (size_t)grid * 2 * 8 * nt;
    return rows * D * 4 + rows * 8 + (size_t)grid * 16;
}

template <int D, int NT, int W, typename T> int launch_clusters(const Args& a, int device, cudaStream_t st) {
    const unsigned segments = (unsigned)(a.B * a.Hkv * a.rts);  // clusters_of bounds them
    constexpr size_t smem = sizeof(Smem<D, NT, W>);
    auto kern = attn_kv8_kernel<D, NT, W, true, T>;
    static std::atomic<unsigned long long> ready{0};  // devices whose limit is raised
    const int rc = raise_smem(kern, smem, device, ready);
    if (rc != B200LAB_OK) return rc;
    return kv8_launch_clusters(1 << a.log2C, kern, dim3(segments << a.log2C), 32 * W, smem, st, a);
}

template <int D, int NT, int W, typename T>
int launch(Args a, void* ws, int grid, int device, cudaStream_t st) {
    const size_t rows = (size_t)grid * 2 * 8 * NT;
    a.part = static_cast<float*>(ws);
    a.meta = reinterpret_cast<int*>(a.part + rows * D + rows * 2);
    constexpr size_t smem = sizeof(Smem<D, NT, W>);
    auto kern = attn_kv8_kernel<D, NT, W, false, T>;
    static std::atomic<unsigned long long> ready{0};  // devices whose limit is raised
    int rc = raise_smem(kern, smem, device, ready);
    if (rc != B200LAB_OK) return rc;
    rc = kv8_launch(kern, dim3(grid), 32 * W, smem, st, a);
    if (rc != B200LAB_OK) return rc;
    const long long used = (long long)a.group * a.max_seqlen_q;
    const int rows_used = (int)(used < 8 * NT ? used : 8 * NT);
    const long long segments = (long long)a.B * a.Hkv * ((used + 8 * NT - 1) / (8 * NT));
    if (segments * 16 >= grid)
        return kv8_launch(attn_kv8_join_kernel<D, NT, T, false>, dim3(grid, (rows_used + 7) / 8), 256, 0, st, a, grid);
    return kv8_launch(attn_kv8_join_kernel<D, NT, T, true>, dim3((unsigned)segments, rows_used), 512, 0, st, a, grid);
}

template <int D, int NT, typename T>
int launch_warps(int warps, const Args& a, void* ws, int grid, int device, cudaStream_t st) {
    if (a.log2C >= 0)
        return warps == kWideWarps ? launch_clusters<D, NT, kWideWarps, T>(a, device, st)
                                   : launch_clusters<D, NT, kMostWarps, T>(a, device, st);
    return warps == 1 ? launch<D, NT, 1, T>(a, ws, grid, device, st) : launch<D, NT, 4, T>(a, ws, grid, device, st);
}

template <typename T>
int launch_d(int D, int nt, int warps, const Args& a, void* ws, int grid, int device, cudaStream_t st) {
    if (D == 256) return launch_warps<256, 1, T>(warps, a, ws, grid, device, st);
    if (D == 128)
        return nt == 1 ? launch_warps<128, 1, T>(warps, a, ws, grid, device, st)
                       : launch_warps<128, 2, T>(warps, a, ws, grid, device, st);
    return nt == 1 ? launch_warps<64, 1, T>(warps, a, ws, grid, device, st)
                   : launch_warps<64, 2, T>(warps, a, ws, grid, device, st);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace b200

B200_DEFINE_ERR_TAKER(attn_kv8, b200::g_err_attn_kv8)

extern "C" size_t attn_fwd_sm100_kv8_workspace(int Hq, int Hkv, int max_seqlen_q, int D) {
    if (Hq < 1 || Hkv < 1 || Hq % Hkv || max_seqlen_q < 1 || (D != 64 && D != 128 && D != 256)) return 0;
    const long long rows = (long long)(Hq / Hkv) * max_seqlen_q;
    const int nt = b200::column_tiles(rows < 64 ? (int)rows : 64, D);
    return b200::workspace_bytes(D, nt, b200::plan_grid(D, nt, 1, b200::device_sm_count()));
}

extern "C" int attn_fwd_sm100_kv8(const void* Q, long long q_stride_token, long long q_stride_head, const void* G,
                                  long long g_stride_token, long long g_stride_head, const void* k_cache,
                                  const void* v_cache, const float* k_scale, const float* v_scale,
                                  const int* block_table, const int* seq_lens, const int* cu_seqlens_q,
                                  int max_seqlen_q, int total_q, void* O, int B, int max_blocks, int n_blocks,
                                  int block_size, int Hq, int Hkv, int D, float scale, int causal, int dtype,
                                  void* workspace, size_t ws_bytes, void* stream) {
    using namespace b200;
    if (!Q || !O || !seq_lens) return B200LAB_ERR_INVALID;
    int rc = kv8_check_cache(k_cache, v_cache, k_scale, v_scale, block_table, B, max_blocks, n_blocks, block_size, Hkv, D);
    if (rc != B200LAB_OK) return rc;
    if (Hq < 1 || Hq % Hkv || max_seqlen_q < 1 || total_q < 1) return B200LAB_ERR_INVALID;
    if (!cu_seqlens_q && (max_seqlen_q != 1 || total_q != B)) return B200LAB_ERR_INVALID;
    if (dtype != B200LAB_F16 && dtype != B200LAB_BF16) return B200LAB_ERR_INVALID;
    if (causal != 0 && causal != 1) return B200LAB_ERR_INVALID;
    if (!(scale > 0.f) || scale > 3.402823466e38f) return B200LAB_ERR_INVALID;
    if (!aligned16(Q) || !aligned16(O) || !aligned16(workspace)) return B200LAB_ERR_INVALID;
    if (q_stride_token < 0 || q_stride_head < 0 || q_stride_token % 8 || q_stride_head % 8) return B200LAB_ERR_INVALID;
    if (G && (g_stride_token < 0 || g_stride_head < 0)) return B200LAB_ERR_INVALID;
    const int most = max_seqlen_q < total_q ? max_seqlen_q : total_q;
    const long long rows = (long long)(Hq / Hkv) * most;
    if (rows > 0xffffffLL) return B200LAB_ERR_UNSUPPORTED;  // 24 bits in a segment's description
    const int nt = column_tiles((int)rows, D);
    const Kv8Device dev = kv8_device();
    const int sms = dev.sms > 0 ? dev.sms : device_sm_count();
    const int rts = (int)((rows + 8 * nt - 1) / (8 * nt));
    const long long segments = (long long)B * Hkv * rts, tokens = (long long)max_blocks * block_size;
    const Clusters clusters = clusters_of(segments, tokens, D, nt, sms);
    const int warps = clusters.log2C >= 0 ? clusters.warps : warps_of(segments, tokens, D, nt, sms);
    const int grid = plan_grid(D, nt, warps, sms);
    if (!workspace || ws_bytes < workspace_bytes(D, nt, plan_grid(D, nt, 1, sms))) return B200LAB_ERR_WORKSPACE;
    if (dev.status != B200LAB_OK) return dev.status;
    Args a;
    a.q = Q, a.g = G, a.o = O;
    a.q_st = q_stride_token, a.q_sh = q_stride_head, a.g_st = g_stride_token, a.g_sh = g_stride_head;
    a.g_aligned = aligned16(G) && g_stride_token % 8 == 0 && g_stride_head % 8 == 0;
    a.k = static_cast<const uint8_t*>(k_cache), a.v = static_cast<const uint8_t*>(v_cache);
    a.table = block_table, a.lens = seq_lens, a.cu = cu_seqlens_q;
    a.k_scale = k_scale, a.v_scale = v_scale;
    a.max_seqlen_q = most, a.total_q = total_q, a.B = B, a.max_blocks = max_blocks, a.n_blocks = n_blocks;
    a.log2P = kv8_log2_block(block_size), a.Hq = Hq, a.Hkv = Hkv, a.group = Hq / Hkv, a.causal = causal;
    a.scale = scale;
    a.rts = rts;
    a.log2C = clusters.log2C;
    a.head_bytes = (uint32_t)(block_size * D);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == B200LAB_F16 ? launch_d<__half>(D, nt, warps, a, workspace, grid, dev.ordinal, st)
                                : launch_d<__nv_bfloat16>(D, nt, warps, a, workspace, grid, dev.ordinal, st);
}
