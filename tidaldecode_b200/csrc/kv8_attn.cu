// One decode step of attention over an 8-bit KV pool, on the tensor cores (mma.sync m16n8k16, fp16 operands).
//
// The mathematics.  A cached element is code * 2^e with one e per (block of slots, head), so e4m3 codes go into the
// products as fp16 values (exactly: fp16 holds every e4m3 value) and the scales stay outside:
//     x_j = (q . k_j) 2^(ek_j) sm log2(e)                       logits in log2 units
//     l   = sum_j 2^(x_j - m)                                   m >= all x_j so far
//     O   = sum_j 2^(x_j + ev_j - M) v_j                        M >= all x_j + ev_j so far
// The value scale goes into the exponent of the weight that the product with V uses, and that weight has a maximum of its
// own: a token of great weight and tiny values does not push the others' weights out of fp16.  m and M are rounded up
// to integers, so x - m and x + ev - M are single roundings and rescaling multiplies by exact powers of two.
//
// Rounding choices.  q is scaled by a power of two so that its largest element lies in [2^11, 2^12): fp16 then holds
// bf16 and fp16 rows exactly (elements 2^25 below the largest lose bits); fp32 rows are split into two fp16 terms (22
// bits).  Weights are scaled to at most 2^14 and enter the product as two fp16 terms, the second the remainder of the first: one
// term alone (half a step is 2^-12) turned every fifteenth bf16 result of a short list to the neighbouring number.  Up to
// four query heads to a unit leave half of the product's eight columns free: they hold the second terms (the free columns
// mirror the queries, so that a lane forms a remainder from logits of its own), times 2^12, and the sums are joined when the
// list ends.  A weight then has 22 bits down to 2^-28 of the heaviest, and tokens down to 2^-50 of it count.  With more
// heads the second terms are a product of their own: for fp32 results times 2^12 as well, against values times 2^-12 (e4m3
// values are multiples of 2^-9 of four bits: exact); for 16-bit results as they are, 11 bits at 2^-28 and an end at 2^-38,
// which such results do not show and which saves 5 % of a long batch.  64 sequences of up to 32 K tokens, 32/8 heads of 128,
// bf16: 138 us with one term, 148 with a second product, 142 with the columns.
// Accumulators, maxima and sums are fp32.  The tensor cores cut a sum's last bits off, and over a long chain that adds up (to
// 8e-6 of a result after 30 K tokens, 1.7e-5 after 7 K tokens to a warp).  So where the result is fp32 the chain is short, and
// what it gives is added by ordinary additions: after every tile where registers allow, after kKv8Chain tiles, with
// the sums in local memory, where they do not (D = 128, up to eight heads to a unit).  8 sequences, one head to a unit, 8192
// tokens, D = 128: 38.7 us unsplit, 43.1 after every tile (spills), 38.8 parked; 16 heads to a unit, 16384 tokens, D = 64: 28.0,
// 28.4, 31.4.  For 16-bit results the rounding of the result is a hundred times larger, and the chain stays whole.
//
// Data movement.  Every warp has a ring of tiles of its own in shared memory, filled with cp.async, 16 bytes to a lane and a
// whole row to adjacent lanes (with the two pieces of a 32-byte sector four lanes apart, sectors were fetched twice: 6.0
// TB/s left L2 for 4.0 TB/s of cache).  No barrier beyond the warp's own, no register held by data in flight.  The order of
// the contraction index and of the output elements is free as long as both operands agree, so the fragments are read
// 16 bytes at a time, from 16-byte pieces that are permuted within 128 bytes so that no two lanes of an access meet
// in a bank.  With lane = 4 g + t, a tile of 16 tokens:
//     S^T = K Q^T      (M = 16 tokens, N = 8 heads): lane reads 16-byte pieces t and 4 + t of K rows g and 8 + g; the four
//                      bytes of a word are elements 2t, 2t+1, 2t+8, 2t+9 of a k-step
//     O^T = V^T P^T    (M = 16 elements, N = 8 heads): lane reads bytes g*D/8.. of V rows 2t, 2t+1, 2t+8, 2t+9; P^T is the
//                      accumulator of S^T transposed in 8 x 8 blocks (movmatrix)
// Both products have the few query heads as N: with heads as M (16 rows, most of them zero) the first took twice the
// instructions and twice the registers.  A lane's accumulators belong to heads 2t and 2t+1 throughout.
//
// Bound by HBM on long contexts: 64 sequences of 16 K tokens, 32/8 heads of 128 (2.1 GB) 334 us, 6.5 TB/s; 16 of them 95 us
// (5.7 TB/s), of which 6 to 8 us pass before the first tile is there, 16 between the first and the last CTA's end and 5 in the
// merge.
// The same tile loop on the tensor cores' 5th-generation instructions has no use here: at most 16 query rows share a K tile
// (a tile of tcgen05.mma has 64), and removing either product altogether takes nothing off (95 us: 94) or, of 32 K tokens with
// logits, 4 of 58 us.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "kv8.cuh"

namespace tidal {

constexpr int kKv8Warps = 8;
constexpr int kKv8Chain = 16;               // tiles whose values tensor cores add up before their sum is parked
constexpr int kKv8Tile = 16;             // tokens a warp takes at a time; it looks them up two tiles at a time
constexpr int kKv8Pair = 2 * kKv8Tile;
constexpr float kLn2 = 0.69314718055994531f;
constexpr int kKv8MaxPrefix = 2048;      // lists whose lengths a CTA adds up itself; beyond, a CTA per list
// Lists up to this long go to a CTA each.  One sequence of 256 / 512 / 1024 tokens, 8 KV heads: 6.5 / 8.8 / 13.0 us that way, 8.6 /
// 8.6 / 9.0 us in ranges and a merge.
constexpr int kKv8SoloTokens = 384;

struct AttnKv8Params {
    const void* q;
    void* o;
    const uint8_t* kv;
    const uint8_t* scales;
    SlotMap map;
    const int32_t* seq_lens;
    int32_t seq_len;
    const int32_t* sel_idx;
    int32_t sel_rows, sel_count;
    int64_t sel_stride;
    const int32_t* sel_counts;
    float* scores;
    int64_t score_stride;
    float* lse;
    float* part_o;               // [units][ranges + lists][rows][D]: what a warp has of a list that it shares with others
    float* part_ml;              // [units][ranges + lists][rows][2]
    uint32_t* status;
    int32_t Hq, Hkv, G, block;
    int32_t lists, per_head;     // token lists: one per sequence, or one per (sequence, query head)
    int32_t groups, rows, units; // query heads of a KV head are taken `rows` (at most 16) at a time, in `groups` groups: a unit each
    int32_t HC, slices;          // units per CTA (its warps take them in turn); CTAs along the units
    int32_t ctas, ranges;        // CTAs that share the lists' tokens; ranges of them per unit: ctas * warps / HC
    int32_t solo;                // a CTA per list (and unit): its warps split the list and merge in shared memory
    int32_t ragged;              // lengths are on the device; every CTA adds them up
    int32_t pairs_per_list;      // !ragged
    int32_t page_shift, block_shift;     // -1 where the size is no power of two
    int32_t blocks_per_page;
    float sm_scale;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The product alone.
__device__ __forceinline__ void mma_f16_fresh(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// An 8 x 8 matrix of 16-bit elements, lane (g, t) holding row g, columns 2t and 2t+1, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Four e4m3 codes to two fp16 pairs.
__device__ __forceinline__ void halves_of(uint32_t codes, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// The part of (lo, hi) that `packed` lost, again as fp16, times `up`.
__device__ __forceinline__ uint32_t pack_f16_rest(float lo, float hi, uint32_t packed, float up = 1.f) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed));
    return pack_f16((lo - f.x) * up, (hi - f.y) * up);
}
// An fp16 pair times 2^-12, exact for e4m3 values: multiples of 2^-9 of four bits.
__device__ __forceinline__ uint32_t shift_down(uint32_t x) {
    const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(0x1p-12f));
    return *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ int list_len_kv8(const AttnKv8Params& p, int list) {
    if (p.sel_idx) return p.sel_counts ? max(0, min(p.sel_counts[list], p.sel_count)) : p.sel_count;
    return p.seq_lens ? max(0, min(p.seq_lens[list], p.seq_len)) : p.seq_len;
}

__device__ __forceinline__ int pairs_of_kv8(int len) { return len > 0 ? (len - 1) / kKv8Pair + 1 : 1; }     // an empty list has one empty pair
// prefix[i] = pairs of the lists before list i, for i <= lists, by the whole CTA (256 threads).
__device__ __forceinline__ void add_up_lists(const AttnKv8Params& p, int* prefix, int* scan) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (p.lists + blockDim.x - 1) / blockDim.x, first = tid * per, last = min(first + per, p.lists);
    int sum = 0;
    for (int i = first; i < last; ++i) sum += pairs_of_kv8(list_len_kv8(p, i));
    int incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += y;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int at = incl - sum;
    for (int i = 0; i < warp; ++i) at += scan[i];
    for (int i = first; i < last; ++i) {
        prefix[i] = at;
        at += pairs_of_kv8(list_len_kv8(p, i));
        if (i == p.lists - 1) prefix[p.lists] = at;
    }
    __syncthreads();
}

// More than 8 query heads to a unit at D = 128 take all registers of an SM for one CTA; its ring then takes the whole memory.
template <int D, bool R2>
struct Kv8Ring {
    static constexpr int stages = D == 128 ? (R2 ? 6 : 3) : 5;
    static constexpr int stage_bytes = kKv8Tile * 2 * D;                 // of one warp: K rows, then V rows
    static constexpr size_t bytes = (size_t)kKv8Warps * stages * stage_bytes;
};
// Byte offset of 16-byte piece c of token i's K row / V row within a tile.  Eight lanes of an access (a quarter of a warp,
// or half of one where a lane reads 8 bytes) have to fall into the eight different pieces of 128 bytes: K rows are
// read by two neighbouring tokens and four neighbouring pieces, V rows by four tokens of one parity and 32 bytes.
template <int D>
__device__ __forceinline__ int k_piece(int i, int c) { return D == 128 ? i * 128 + (c ^ (i & 1) * 4) * 16 : i * 64 + c * 16; }
template <int D>
__device__ __forceinline__ int v_piece(int i, int c) {
    if (D == 128) return i * 128 + (c ^ (i & 6)) * 16;
    return (i >> 1) * 128 + ((i ^ i >> 1) & 1) * 64 + (c ^ (i >> 1 & 2)) * 16;
}
// Four consecutive elements of a row.
template <typename T>
__device__ __forceinline__ void load4(const T* p, float* f) {
    if (sizeof(T) == 4) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = to_f32(e[i]);
    }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v) {
    if (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = v;
    } else {
        alignas(8) const T e[4] = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
        *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
    }
}

// 2^e as two factors, e an integer of at most 127.  One factor alone becomes zero below 2^-126, where the product with a sum
// (up to 2^14 times as large as what it stands for) need not.
struct Pow2 {
    float a, b;
    __device__ __forceinline__ explicit Pow2(float e) {
        const int k = (int)fmaxf(e, -250.f), h = k >> 1;
        a = __uint_as_float((uint32_t)(127 + h) << 23);
        b = __uint_as_float((uint32_t)(127 + k - h) << 23);
    }
    __device__ __forceinline__ float times(float x) const { return x * a * b; }
};

// Softmax statistics and output of one query head to their final form.
__device__ __forceinline__ float attn_kv8_lse(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2; }

// Which of `ranges` equal ranges of `total` items holds item i, and where range r begins.  ranges <= total.
__device__ __forceinline__ int range_begin(int r, int total, int ranges) { return (int)((int64_t)r * total / ranges); }
__device__ __forceinline__ int range_of(int i, int total, int ranges) { return (int)((((int64_t)i + 1) * ranges - 1) / total); }

// Work is dealt out in pairs of tiles, 32 tokens.  Laid end to end, the pairs of all token lists are cut into equal ranges, one
// to a warp and unit (KV head, or up to 16 query heads of one), whatever list they fall into: a batch of very different
// lengths keeps every SM busy to the end.  A warp keeps its ring full across the lists' borders and waits for no other
// warp; where a list is shared, each leaves a partial (o relative to m, m, l) and merge_kv8_kernel adds them in order.
// The order of additions depends on the lengths and the launch alone.  Short lists go the other way (solo): one CTA per
// list and unit, whose warps merge through shared memory, with no second launch.
template <typename T, int D, int H>      // H: query heads to a unit, at most: 4, 8 or 16
__global__ void __launch_bounds__(kKv8Warps * 32, H == 16 && (sizeof(T) == 4 || D == 128) ? 1 : 2) attn_kv8_kernel(const __grid_constant__ AttnKv8Params p) {
    constexpr bool QS = sizeof(T) == 4, R2 = H == 16, MIRROR = H == 4;
    constexpr float kBinades = QS ? 0.f : 14.f;                          // of the weights' range that M leaves to the exponent
    constexpr int S = Kv8Ring<D, R2>::stages, KC = D / 64, KS = D / 16, VB = D / 8, NR = R2 ? 2 : 1;
    constexpr bool park = QS && D == 128 && !R2;
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int NP = S <= 4 ? 2 : 4;       // pairs of tiles whose scales are kept: a slot is refilled S - 2 NP <= 0 tiles after its last use
    // per token: scale of K (-1: no token) and exponent of the scale of V (-inf: the block reads as zeros)
    __shared__ __align__(16) float2 sc_ring[kKv8Warps][NP][2 * kKv8Tile];
    __shared__ float ml[kKv8Warps][16][2];
    __shared__ int s_scan[kKv8Warps];
    int* prefix = reinterpret_cast<int*>(smem + Kv8Ring<D, R2>::bytes);      // [lists + 1] when the lengths are added up here

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int TG = kKv8Warps / p.HC, uw = warp % p.HC, tg = warp / p.HC;
    const int cta = (int)(blockIdx.x / (uint32_t)p.slices), slice = (int)(blockIdx.x - (uint32_t)cta * (uint32_t)p.slices);
    unsigned char* ring = smem + (size_t)warp * S * Kv8Ring<D, R2>::stage_bytes;
    if (tid == 0) TIDAL_STAMP(0);
    pdl_wait();
    pdl_launch_dependents();
    if (tid == 0) TIDAL_STAMP(1);

    // ---- this warp's range [t0, t1) of pairs
    int t0, t1, list = 0, first = 0;                                     // `list` starts at pair `first`
    if (p.solo) {
        list = cta;
        const int n = pairs_of_kv8(list_len_kv8(p, list));
        t0 = range_begin(tg, n, TG);
        t1 = range_begin(tg + 1, n, TG);
    } else {
        int total;
        if (p.ragged) {
            add_up_lists(p, prefix, s_scan);
            total = prefix[p.lists];
        } else {
            total = p.pairs_per_list * p.lists;
        }
        const int ranges = min(p.ranges, total), r = cta * TG + tg;      // no range without a pair: every part that is added exists
        if (r >= ranges) return;
        t0 = range_begin(r, total, ranges);
        t1 = range_begin(r + 1, total, ranges);
        if (p.ragged) {
            int hi = p.lists;                                            // last list that starts at or before t0
            while (hi - list > 1) {
                const int mid = (list + hi) >> 1;
                if (prefix[mid] <= t0) list = mid; else hi = mid;
            }
            first = prefix[list];
        } else {
            list = t0 / p.pairs_per_list;
            first = list * p.pairs_per_list;
        }
    }
    const int unit = slice * p.HC + uw;

    // ---- where a list's tokens and heads are
    struct List {
        int list, first, next;           // pairs [first, next)
    };
    auto enter = [&](List& w, int i, int at) -> int {
        const int len = list_len_kv8(p, i);
        w.list = i;
        w.first = at;
        w.next = at + pairs_of_kv8(len);
        return len;
    };
    const int unit_kvh = unit / p.groups, unit_hq = unit_kvh * p.G + (unit - unit_kvh * p.groups) * p.rows;
    auto seq_of = [&](int i) -> int { return p.per_head ? i / p.Hq : i; };                          // sequence of a list
    auto kvh_of = [&](int i) -> int { return p.per_head ? i % p.Hq / p.G : unit_kvh; };
    auto row_of = [&](int i) -> size_t { return p.per_head ? (size_t)i : (size_t)i * p.Hq + unit_hq; };     // row of its first query head
    const int heads = p.per_head ? 1 : min(p.rows, (unit_kvh + 1) * p.G - unit_hq);                // query heads of the unit

    // ---- looking tokens up: lane i follows token i of a pair; its list entry is loaded two pairs ahead of its copies, its
    //      page one pair ahead, its scales with the copies
    constexpr int PR = D / 16, TI = 32 / PR;                              // 16-byte pieces of a row; tokens that one copy of the warp covers
    const int c_tok = lane / PR, c_piece = lane % PR;
    const int ps = p.map.page_size;
    const uint32_t pitch = (uint32_t)p.Hkv * D;
    const uint32_t ring_k = smem_u32(ring) + k_piece<D>(c_tok, c_piece), ring_v = smem_u32(ring) + kKv8Tile * D + v_piece<D>(c_tok, c_piece);
    const int k_off = k_piece<D>(g, t), v_off = v_piece<D>(2 * t, g * VB / 16) + (g * VB & 15);
    const int v_off1 = v_piece<D>(2 * t + 1, g * VB / 16) + (g * VB & 15);
    const uint32_t sc_plane = (uint32_t)p.blocks_per_page * p.Hkv;
    List ahead_l;                                                        // of the pair whose entries are loaded next
    int ahead_t = t0, ahead_len = enter(ahead_l, list, first);
    auto fetch_pos = [&]() -> int {
        const int i = (ahead_t - ahead_l.first) * kKv8Pair + lane;
        if (ahead_t >= t1 || i >= ahead_len) return INT_MIN;             // no token here
        return p.sel_idx ? max(p.sel_idx[(size_t)ahead_l.list * p.sel_stride + i], -1) : i;
    };
    auto step_ahead = [&]() {
        ++ahead_t;
        if (ahead_t == ahead_l.next && ahead_t < t1) ahead_len = enter(ahead_l, ahead_l.list + 1, ahead_t);
    };
    auto page_of = [&](int pos) -> int { return p.page_shift >= 0 ? pos >> p.page_shift : pos / ps; };
    auto fetch_page = [&](int pos, int i) -> int {
        const int b = seq_of(i);
        if (p.sel_idx && pos >= (p.seq_lens ? min(p.seq_lens[b], p.seq_len) : p.seq_len)) return -1;
        if (pos < 0) return -1;
        return p.map.page_table ? p.map.page_table[(size_t)b * p.map.pt_stride + page_of(pos)] : (int)((int64_t)b * p.map.pt_stride) + page_of(pos);
    };
    int list_c = ahead_l.list, pos_c = fetch_pos(), page_c = fetch_page(pos_c, list_c);            // the pair to be copied next
    step_ahead();
    int list_n = ahead_l.list, pos_n = fetch_pos();                                                // the one behind it
    step_ahead();
    int row = -1;                                                        // pool row of the lane's K row (its V row lies ps rows further), or -1
    uint32_t sc_k = 0, sc_v = 0;                                         // its scale bytes
    uint32_t head_off = 0;                                               // byte offset of its head (and the lane's piece) in a row
    uint32_t full = 0, half = 0;     // bit i, of the pair copied i pairs ago: every token is there; a token of its second tile is there
    auto look_up = [&]() {
        row = -1;
        const uint32_t kvh = (uint32_t)kvh_of(list_c);
        if (page_c >= 0 && page_c < (int)p.map.num_pages) {
            const int entry = pos_c - page_of(pos_c) * ps;
            row = page_c * 2 * ps + entry;
            uint32_t at = (uint32_t)page_c * 2u * sc_plane + kvh;              // scale bytes number less than 2^32, checked on the host
            if (p.blocks_per_page > 1) at += (uint32_t)(p.block_shift >= 0 ? entry >> p.block_shift : entry / p.block) * (uint32_t)p.Hkv;
            sc_k = p.scales[at];
            sc_v = p.scales[at + sc_plane];
        } else if (pos_c != INT_MIN) {
            atomicOr(p.status, TIDAL_DEV_BAD_INDEX);
        }
        const uint32_t there = __ballot_sync(0xffffffffu, row >= 0);
        full = full << 1 | (there == 0xffffffffu ? 1u : 0u);
        half = half << 1 | (there >> kKv8Tile ? 1u : 0u);
        head_off = kvh * D + c_piece * 16;
        page_c = fetch_page(pos_n, list_n);
        pos_c = pos_n;
        list_c = list_n;
        pos_n = fetch_pos();
        list_n = ahead_l.list;
        step_ahead();
    };
    auto park_scales = [&](int pair) {
        sc_ring[warp][pair & (NP - 1)][lane] = row >= 0 ? make_float2(scale_value(sc_k), sc_v ? (float)((int)sc_v - 127) : -INFINITY) : make_float2(-1.f, -INFINITY);
    };
    auto copy = [&](int it, uint32_t slot) {
        if ((it & 1) && !(half & 1u)) return;
        const int l0 = (it & 1) * kKv8Tile + c_tok;
        const uint8_t *k_src = p.kv + head_off, *v_src = k_src + (size_t)ps * pitch;
        if (full & 1u) {
#pragma unroll
            for (int i = 0; i < kKv8Tile / TI; ++i) {
                const uint32_t r = (uint32_t)__shfl_sync(0xffffffffu, row, l0 + i * TI);
                cp_async16(ring_k + slot + i * 512, k_src + (uint64_t)r * pitch);
                cp_async16((D == 128 && (i & 1) ? ring_v ^ 64u : ring_v) + slot + i * 512, v_src + (uint64_t)r * pitch);
            }
        } else {
#pragma unroll
            for (int i = 0; i < kKv8Tile / TI; ++i) {
                const int r = __shfl_sync(0xffffffffu, row, l0 + i * TI);
                const uint64_t at = (uint64_t)max(r, 0) * pitch;
                cp_async16_or_zero(ring_k + slot + i * 512, k_src + at, r >= 0);
                cp_async16_or_zero((D == 128 && (i & 1) ? ring_v ^ 64u : ring_v) + slot + i * 512, v_src + at, r >= 0);
            }
        }
    };

    const int n_it = 2 * (t1 - t0);                                      // tiles (the second of a pair may be empty)
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
        if (s < n_it) {
            if ((s & 1) == 0) {
                look_up();
                park_scales(s >> 1);
            }
            copy(s, s * Kv8Ring<D, R2>::stage_bytes);
        }
        cp_async_commit();
    }
    uint32_t put_slot = (S - 1) * Kv8Ring<D, R2>::stage_bytes, use_slot = 0;

    List cur;                                                            // of the tile being computed
    (void)enter(cur, list, first);
    bool fresh = true;                                                   // a list begins: its queries are to be loaded
    uint32_t qa[NR][KS][2], ql[QS ? NR : 1][QS ? KS : 1][2];             // Q fragments (lane: head g of each eight), scaled to [2^11, 2^12) per head
    float qn2[NR][2];                                                    // of heads 2t, 2t+1: undoes the scaling, applies sm_scale, in log2 units
    float o[NR][KS][4];                                                  // [eight heads][16 elements]: elements 2j, 2j+1 of g*D/8.., heads 2t, 2t+1
    float m[NR][2], M[NR][2], l[NR][2];
    volatile float parked[NR * KS * 4];                                  // sums of earlier tiles of the list
    bool any_parked = false;
    auto unpark = [&]() {
        if (!park || !any_parked) return;
#pragma unroll
        for (int i = 0; i < NR * KS * 4; ++i) o[i / (4 * KS)][i / 4 % KS][i % 4] += parked[i];
    };
    // MIRROR: what the second terms gave, in the columns of heads 4 to 7, is added to the first terms' sums
    auto fold = [&]() {
        if (!MIRROR) return;
#pragma unroll
        for (int j = 0; j < KS; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[0][j][i] = fmaf(__shfl_xor_sync(0xffffffffu, o[0][j][i], 2), 0x1p-12f, o[0][j][i]);
    };
    for (int it = 0; it < n_it || (p.solo && fresh); ++it) {
        const int ahead = it + S - 1;
        const bool looked = ahead < n_it && (ahead & 1) == 0;
        if (looked) look_up();
        if (ahead < n_it) copy(ahead, put_slot);
        put_slot = put_slot == (S - 1) * Kv8Ring<D, R2>::stage_bytes ? 0 : put_slot + Kv8Ring<D, R2>::stage_bytes;
        cp_async_commit();
        if (fresh) {
            fresh = any_parked = false;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const int head = MIRROR ? g & 3 : g + 8 * r;
                const T* qrow = reinterpret_cast<const T*>(p.q) + (row_of(cur.list) + (head < heads ? head : 0)) * D;
                float f[KS][4], top = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    load4(qrow + (ks >> 2) * 64 + t * 16 + (ks & 3) * 4, f[ks]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float a = fabsf(f[ks][i]);
                        top = a < INFINITY ? fmaxf(top, a) : top;
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                int sh = 138 - (int)(__float_as_uint(top) >> 23);       // 11 less the exponent of the largest element
                sh = top == 0.f ? 0 : min(sh, 120);
                const float up = __uint_as_float((uint32_t)(127 + sh) << 23);
                const float down = p.sm_scale * __uint_as_float((uint32_t)(127 - sh) << 23);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    qn2[r][e] = __shfl_sync(0xffffffffu, down, 8 * t + 4 * e) * kLog2e;
                    m[r][e] = M[r][e] = -FLT_MAX;
                    l[r][e] = 0.f;
                }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float x0 = f[ks][2 * i] * up, x1 = f[ks][2 * i + 1] * up;
                        qa[r][ks][i] = head < heads ? pack_f16(x0, x1) : 0u;
                        if (QS) ql[QS ? r : 0][QS ? ks : 0][i] = head < heads ? pack_f16_rest(x0, x1, qa[r][ks][i]) : 0u;
                    }
#pragma unroll
                for (int j = 0; j < KS; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[r][j][i] = 0.f;
            }
            if (n_it == 0) break;                                        // solo: nothing for this warp but an empty share
        } else if (park && it % kKv8Chain == 0) {
            unpark();
#pragma unroll
            for (int i = 0; i < NR * KS * 4; ++i) {
                parked[i] = o[i / (4 * KS)][i / 4 % KS][i % 4];
                o[i / (4 * KS)][i / 4 % KS][i % 4] = 0.f;
            }
            any_parked = true;
        }
        cp_async_wait<S - 1>();
        __syncwarp();
        if (tid == 0 && it == 0) TIDAL_STAMP(2);
        const unsigned char* st = ring + use_slot;
        use_slot = use_slot == (S - 1) * Kv8Ring<D, R2>::stage_bytes ? 0 : use_slot + Kv8Ring<D, R2>::stage_bytes;
        // the pair of tile `it` was looked up this many pairs before the newest one
        const int age = (min(ahead, n_it - 1) >> 1) - (it >> 1);
        if (!(it & 1) || (half >> age & 1u)) {
            const bool all = full >> age & 1u;
            // ---- S^T = K Q^T: tokens g and 8 + g, heads 2t and 2t+1
            float sf[NR][4], sl[QS ? NR : 1][4];                         // the second terms' products have a chain of their own
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) sf[r][i] = sl[QS ? r : 0][i] = 0.f;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const uint4 k0 = *reinterpret_cast<const uint4*>(st + (k_off ^ c * 64)), k1 = *reinterpret_cast<const uint4*>(st + 8 * D + (k_off ^ c * 64));
                const uint32_t lo[4] = {k0.x, k0.y, k0.z, k0.w}, hi[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int ks = c * 4 + i;
                    uint32_t a[4];
                    halves_of(lo[i], a[0], a[2]);
                    halves_of(hi[i], a[1], a[3]);
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        mma_f16(sf[r], a[0], a[1], a[2], a[3], qa[r][ks][0], qa[r][ks][1]);
                        if (QS) mma_f16(sl[QS ? r : 0], a[0], a[1], a[2], a[3], ql[QS ? r : 0][QS ? ks : 0][0], ql[QS ? r : 0][QS ? ks : 0][1]);
                    }
                }
            }
            if (QS) {
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sf[r][i] += sl[QS ? r : 0][i];
            }
            // ---- scales of the two tokens; value i of a lane: token g + 8 (i / 2), head 2t + i % 2
            const float2* scp = &sc_ring[warp][(it >> 1) & (NP - 1)][(it & 1) * kKv8Tile + g];
            const float2 s0 = scp[0], s1 = scp[8];
            const float kf[2] = {s0.x, s1.x}, ev[2] = {s0.y, s1.y};
            if (p.scores) {
                const int i0 = (t0 + (it >> 1) - cur.first) * kKv8Pair + (it & 1) * kKv8Tile + g;      // list index of the lane's first token
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int head = 2 * t + (i & 1) + 8 * r;
                        if (head < heads && kf[i >> 1] >= 0.f)
                            p.scores[(row_of(cur.list) + head) * p.score_stride + i0 + (i >> 1) * 8] = sf[r][i] * (kf[i >> 1] * qn2[r][i & 1]) * kLn2;
                    }
            }
            // ---- exponents of the sums: xl = x - m for the denominator, xw = x + ev - M for the weights.  M is kept less
            //      the 14 binades of the weights' range; where the result is fp32 they are a factor behind the exponential, so
            //      that the argument of a heavy token's is small and rounded finely (2^-21 of a weight otherwise)
            float xl[NR][4], xw[NR][4];
            auto exponents = [&]() -> bool {
                float top = 0.f, topw = kBinades;
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float f = kf[i >> 1] * qn2[r][i & 1];
                        xl[r][i] = fmaf(sf[r][i], f, -m[r][i & 1]);
                        xw[r][i] = fmaf(sf[r][i], f, ev[i >> 1] - M[r][i & 1]);
                    }
                if (!all) {
#pragma unroll
                    for (int r = 0; r < NR; ++r)
#pragma unroll
                        for (int i = 0; i < 4; ++i) xl[r][i] = kf[i >> 1] < 0.f ? -INFINITY : xl[r][i];
                }
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        top = fmaxf(top, xl[r][i]);
                        topw = fmaxf(topw, xw[r][i]);
                    }
                return top > 0.f || topw > kBinades;
            };
            if (__any_sync(0xffffffffu, exponents())) {
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = -FLT_MAX, topv = -FLT_MAX;
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if (kf[i] >= 0.f) {
                                const float x = sf[r][2 * i + e] * (kf[i] * qn2[r][e]);
                                top = fmaxf(top, x);
                                topv = fmaxf(topv, x + ev[i]);
                            }
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) {
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                            topv = fmaxf(topv, __shfl_xor_sync(0xffffffffu, topv, off));
                        }
                        const float mn = fmaxf(m[r][e], ceilf(top)), Mn = fmaxf(M[r][e], ceilf(topv) - kBinades);
                        l[r][e] *= fast_exp2(m[r][e] - mn);
                        const float a = fast_exp2(M[r][e] - Mn);
                        m[r][e] = mn;
                        M[r][e] = Mn;
#pragma unroll
                        for (int j = 0; j < KS; ++j) {
                            o[r][j][e] *= a;
                            o[r][j][2 + e] *= a;
                        }
                        if (park && any_parked) {
#pragma unroll
                            for (int j = 0; j < KS; ++j) {
                                parked[(r * KS + j) * 4 + e] = parked[(r * KS + j) * 4 + e] * a;
                                parked[(r * KS + j) * 4 + 2 + e] = parked[(r * KS + j) * 4 + 2 + e] * a;
                            }
                        }
                    }
                exponents();
            }
            uint32_t pb[NR][2], pl[NR][2];                               // first and second terms (MIRROR: both in pb)
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float w[4];
                l[r][0] += fast_exp2(xl[r][0]) + fast_exp2(xl[r][2]);
                l[r][1] += fast_exp2(xl[r][1]) + fast_exp2(xl[r][3]);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = QS ? fast_exp2(xw[r][i]) * 0x1p14f : fast_exp2(xw[r][i]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t hi = pack_f16(w[2 * i], w[2 * i + 1]);
                    const uint32_t rest = pack_f16_rest(w[2 * i], w[2 * i + 1], hi, QS || MIRROR ? 0x1p12f : 1.f);
                    pb[r][i] = transpose8x8(MIRROR && t >= 2 ? rest : hi);
                    if (!MIRROR) pl[r][i] = transpose8x8(rest);
                }
            }
            // ---- O^T += V^T P^T
            st += kKv8Tile * D;
            uint32_t vw[4][VB / 4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (VB == 16) {
                    const uint4 q4 = *reinterpret_cast<const uint4*>(st + (i >> 1) * 8 * D + (i & 1 ? v_off1 : v_off));
                    vw[i][0] = q4.x, vw[i][1] = q4.y, vw[i][VB / 4 - 2] = q4.z, vw[i][VB / 4 - 1] = q4.w;
                } else {
                    const uint2 q2 = *reinterpret_cast<const uint2*>(st + (i >> 1) * 8 * D + (i & 1 ? v_off1 : v_off));
                    vw[i][0] = q2.x, vw[i][1] = q2.y;
                }
            }
#pragma unroll
            for (int w = 0; w < VB / 4; ++w) {
                uint32_t a[2][4];                                        // [token pair][element of the word], a pair of tokens each
#pragma unroll
                for (int h2 = 0; h2 < 2; ++h2) {
                    halves_of(__byte_perm(vw[2 * h2][w], vw[2 * h2 + 1][w], 0x5140), a[h2][0], a[h2][1]);
                    halves_of(__byte_perm(vw[2 * h2][w], vw[2 * h2 + 1][w], 0x7362), a[h2][2], a[h2][3]);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t low[4] = {a[0][2 * e], a[0][2 * e + 1], a[1][2 * e], a[1][2 * e + 1]};      // operand of the second terms
                    if (QS && !MIRROR) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) low[i] = shift_down(low[i]);
                    }
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        if (QS && !park) {
                            float part[4];
                            if (MIRROR) {
                                mma_f16_fresh(part, a[0][2 * e], a[0][2 * e + 1], a[1][2 * e], a[1][2 * e + 1], pb[r][0], pb[r][1]);
                            } else {
                                mma_f16_fresh(part, low[0], low[1], low[2], low[3], pl[r][0], pl[r][1]);
                                mma_f16(part, a[0][2 * e], a[0][2 * e + 1], a[1][2 * e], a[1][2 * e + 1], pb[r][0], pb[r][1]);
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[r][2 * w + e][i] += part[i];
                            continue;
                        }
                        mma_f16(o[r][2 * w + e], a[0][2 * e], a[0][2 * e + 1], a[1][2 * e], a[1][2 * e + 1], pb[r][0], pb[r][1]);
                        if (!MIRROR) mma_f16(o[r][2 * w + e], low[0], low[1], low[2], low[3], pl[r][0], pl[r][1]);
                    }
                }
            }
        }
        if (looked) park_scales(ahead >> 1);
        __syncwarp();                                                    // the tile's slot is the next to be filled
        // ---- the warp's share of the list ends here
        const int done = t0 + (it >> 1) + 1;
        if (!(it & 1) || (done != cur.next && done != t1) || p.solo) continue;
        unpark();
        fold();
        const bool whole = done == cur.next && t0 <= cur.first;
        const int range = cta * TG + tg;
        const size_t part = ((size_t)unit * (p.ranges + p.lists) + range + cur.list) * p.rows;
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int head = 2 * t + e + 8 * r;
                float sum = l[r][e];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                if (head >= heads) continue;
                Pow2 f(M[r][e] + (kBinades - 14.f) - m[r][e]);
                if (whole) f.b *= sum == 0.f ? 0.f : 1.f / sum;
                const size_t out = row_of(cur.list) + head;
                if (g == 0) {
                    if (!whole) *reinterpret_cast<float2*>(p.part_ml + (part + head) * 2) = make_float2(m[r][e], sum);
                    else if (p.lse) p.lse[out] = attn_kv8_lse(m[r][e], sum);
                }
#pragma unroll
                for (int j = 0; j < KS; j += 2) {
                    const float4 v = make_float4(f.times(o[r][j][e]), f.times(o[r][j][2 + e]), f.times(o[r][j + 1][e]), f.times(o[r][j + 1][2 + e]));
                    if (whole) store4(reinterpret_cast<T*>(p.o) + out * D + g * VB + 2 * j, v);
                    else *reinterpret_cast<float4*>(p.part_o + (part + head) * D + g * VB + 2 * j) = v;
                }
            }
        fresh = true;
        if (done < t1) (void)enter(cur, cur.list + 1, done);
    }
    cp_async_wait<0>();
    if (tid == 0) TIDAL_STAMP(3);
    if (!p.solo) return;

    // ---- solo: the warps of a unit merge through shared memory, o relative to m
    unpark();
    fold();
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);                          // [warps][rows][D]
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int head = 2 * t + e + 8 * r;
            float sum = l[r][e];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            if (head >= heads) continue;
            if (g == 0) {
                ml[warp][head][0] = m[r][e];
                ml[warp][head][1] = sum;
            }
            const Pow2 f(M[r][e] + (kBinades - 14.f) - m[r][e]);
            float* at = so + ((size_t)warp * p.rows + head) * D + g * VB;
#pragma unroll
            for (int j = 0; j < KS; ++j) *reinterpret_cast<float2*>(at + 2 * j) = make_float2(f.times(o[r][j][e]), f.times(o[r][j][2 + e]));
        }
    __syncthreads();
    for (int i = tid; i < heads * (D / 4); i += blockDim.x) {            // one unit to a CTA
        const int head = i / (D / 4), d = (i - head * (D / 4)) * 4;
        float mx = -FLT_MAX, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kKv8Warps; ++w) mx = fmaxf(mx, ml[w][head][0]);
#pragma unroll
        for (int w = 0; w < kKv8Warps; ++w) {
            const Pow2 f(ml[w][head][0] - mx);
            const float4 v = *reinterpret_cast<const float4*>(so + ((size_t)w * p.rows + head) * D + d);
            sum += f.times(ml[w][head][1]);
            acc.x = fmaf(f.a * v.x, f.b, acc.x);
            acc.y = fmaf(f.a * v.y, f.b, acc.y);
            acc.z = fmaf(f.a * v.z, f.b, acc.z);
            acc.w = fmaf(f.a * v.w, f.b, acc.w);
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const size_t out = row_of(cur.list) + head;
        store4(reinterpret_cast<T*>(p.o) + out * D + d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
        if (p.lse && d == 0) p.lse[out] = attn_kv8_lse(mx, sum);
    }
    if (tid == 0) TIDAL_STAMP(4);
}

// Adds up the parts of the lists that several warps shared, in the order of their tokens.  A CTA takes `8 / split` query
// heads, `split` warps to a head; where there are few heads only blockIdx.y's 32 elements of them, four parts to a warp at a
// time (one list of 256 K tokens: 10 us less).  What depends on lengths and launch alone is worked out before the attention
// kernel has ended; then a part costs one trip to L2: each group of lanes keeps a maximum of its own.  (The lengths were
// there before that kernel began: it waits for its predecessor before it lets this one start.)  Bound by latency: done 3
// to 5 us after the last CTA of the attention kernel (7 where 64 ragged sequences' lengths are added up), 7.5 us alone and cold.
template <typename T, int D>
__global__ void __launch_bounds__(256) merge_kv8_kernel(const __grid_constant__ AttnKv8Params p, int split) {
    extern __shared__ int prefix_m[];                    // [lists + 1], ragged
    __shared__ float4 sh_o[8][D / 4];                    // by type on 16 bytes
    __shared__ float sh_ml[8][2];
    __shared__ int s_scan[8];
    if (threadIdx.x == 0) TIDAL_STAMP(8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane >> 3, d = (lane & 7) * 4;
    const int per_cta = 8 / split, member = warp % split;
    const int64_t head_id = (int64_t)blockIdx.x * per_cta + warp / split;        // list-major: (list, query head of the list)
    const int per_list = p.per_head ? 1 : p.Hq;
    const bool live = head_id < (int64_t)p.lists * per_list;
    const int list = live ? (int)(head_id / per_list) : 0, h = live ? (int)(head_id - (int64_t)list * per_list) : 0;
    if (p.ragged) add_up_lists(p, prefix_m, s_scan);
    const int total = p.ragged ? prefix_m[p.lists] : p.pairs_per_list * p.lists;
    const int begin = p.ragged ? prefix_m[list] : list * p.pairs_per_list, end = p.ragged ? prefix_m[list + 1] : begin + p.pairs_per_list;
    const int ranges = min(p.ranges, total);
    const int r0 = range_of(begin, total, ranges), parts = range_of(end - 1, total, ranges) - r0 + 1;
    const int kvh = h / p.G, in_kvh = h - kvh * p.G;
    const int unit = p.per_head ? 0 : kvh * p.groups + in_kvh / p.rows, head = p.per_head ? 0 : in_kvh % p.rows;
    const size_t part = ((size_t)unit * (p.ranges + p.lists) + r0 + list) * p.rows + head;
    const float2* part_ml = reinterpret_cast<const float2*>(p.part_ml) + part;
    const size_t out = p.per_head ? (size_t)list : (size_t)list * p.Hq + h;
    const bool work = live && parts > 1;
    pdl_wait();
    pdl_launch_dependents();
    if (threadIdx.x == 0) TIDAL_STAMP(9);
    // the four groups of eight lanes take four parts of one 32-element chunk, or (gridDim.y == 1) the chunks of a head
    const int chunks = gridDim.y == 1 ? D / 32 : 1, groups = 4 / chunks;
    const int chunk = sub % chunks, place = sub / chunks;
    const int at = (blockIdx.y + chunk) * 32 + d;
    const float* part_o = p.part_o + part * D + at;
    float mx = -FLT_MAX, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto rescale = [&](float to) {
        const Pow2 f(mx - to);
        mx = to;
        sum = f.times(sum);
        acc.x = f.times(acc.x), acc.y = f.times(acc.y), acc.z = f.times(acc.z), acc.w = f.times(acc.w);
    };
    auto add = [&](float m, float l, float4 v) {
        const Pow2 f(m - mx);
        sum += f.times(l);
        acc.x = fmaf(f.a * v.x, f.b, acc.x);
        acc.y = fmaf(f.a * v.y, f.b, acc.y);
        acc.z = fmaf(f.a * v.z, f.b, acc.z);
        acc.w = fmaf(f.a * v.w, f.b, acc.w);
    };
    constexpr int K = 4;                                 // parts of a group in flight
    const int stride = split * groups;
    for (int k0 = member * groups + place; work && k0 < parts; k0 += stride * K) {
        float2 s[K];
        float4 v[K];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int k = k0 + i * stride;
            s[i] = make_float2(-FLT_MAX, 0.f);
            v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k < parts) {
                s[i] = part_ml[(size_t)k * p.rows];
                v[i] = *reinterpret_cast<const float4*>(part_o + (size_t)k * p.rows * D);
            }
        }
        rescale(fmaxf(fmaxf(mx, fmaxf(s[0].x, s[1].x)), fmaxf(s[2].x, s[3].x)));
#pragma unroll
        for (int i = 0; i < K; ++i) add(s[i].x, s[i].y, v[i]);
    }
    float top = mx;
    for (int off = 8 * chunks; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    rescale(top);
    for (int off = 8 * chunks; off < 32; off <<= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, off);
        acc.x += __shfl_xor_sync(0xffffffffu, acc.x, off);
        acc.y += __shfl_xor_sync(0xffffffffu, acc.y, off);
        acc.z += __shfl_xor_sync(0xffffffffu, acc.z, off);
        acc.w += __shfl_xor_sync(0xffffffffu, acc.w, off);
    }
    if (split > 1) {
        if (place == 0) sh_o[warp][(chunk * 32 + d) / 4] = acc;
        if (lane == 0) sh_ml[warp][0] = mx, sh_ml[warp][1] = sum;
        __syncthreads();
        if (member == 0 && place == 0) {
            for (int w = 1; w < split; ++w) top = fmaxf(top, sh_ml[warp + w][0]);
            rescale(top);
            for (int w = 1; w < split; ++w) add(sh_ml[warp + w][0], sh_ml[warp + w][1], sh_o[warp + w][(chunk * 32 + d) / 4]);
        }
    }
    if (work && member == 0 && place == 0) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        store4(reinterpret_cast<T*>(p.o) + out * D + at, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
        if (p.lse && lane == 0 && blockIdx.y == 0) p.lse[out] = attn_kv8_lse(mx, sum);
    }
    if (threadIdx.x == 0) TIDAL_STAMP(10);
}

template <typename T, int D, int H>
static int launch_one_kv8(const AttnKv8Params& p, cudaStream_t st) {
    constexpr bool R2 = H == 16;
    const size_t smem = Kv8Ring<D, R2>::bytes + (p.ragged && !p.solo ? sizeof(int) * (p.lists + 1) : 0);
    // the limit is set to the most that a call may need, once per device (the call costs half a microsecond)
    static std::atomic<uint64_t> set{0};
    int dev = 0;
    TIDAL_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !(set.load(std::memory_order_relaxed) >> dev & 1u)) {
        TIDAL_CUDA_OK(cudaFuncSetAttribute(attn_kv8_kernel<T, D, H>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)(Kv8Ring<D, R2>::bytes + sizeof(int) * (kKv8MaxPrefix + 1))));
        if (dev < 64) set.fetch_or((uint64_t)1 << dev);
    }
    TIDAL_CUDA_OK(launch_pdl(attn_kv8_kernel<T, D, H>, dim3((unsigned)p.slices * (unsigned)p.ctas), dim3(kKv8Warps * 32), smem, st, 1, p));
    count_launch();
    return TIDAL_OK;
}
template <typename T, int D>
static int launch_attn_kv8(const AttnKv8Params& p, cudaStream_t st) {
    const int rc = p.rows > 8 ? launch_one_kv8<T, D, 16>(p, st) : p.rows > 4 ? launch_one_kv8<T, D, 8>(p, st) : launch_one_kv8<T, D, 4>(p, st);
    if (rc != TIDAL_OK || p.solo || p.ranges == 1) return rc;
    const int64_t heads = (int64_t)p.lists * (p.per_head ? 1 : p.Hq);
    const int split = p.ranges >= 16 * (int64_t)p.lists ? 8 : p.ranges >= 4 * (int64_t)p.lists ? 4 : 1;
    const unsigned ctas = (unsigned)((heads + 8 / split - 1) / (8 / split));
    TIDAL_CUDA_OK(launch_pdl(merge_kv8_kernel<T, D>, dim3(ctas, ctas <= (unsigned)sm_count_cached() ? D / 32 : 1), dim3(256),
                             p.ragged ? sizeof(int) * (p.lists + 1) : 0, st, 1, p, split));
    count_launch();
    return TIDAL_OK;
}

}  // namespace tidal

using namespace tidal;

extern "C" int tidal_decode_attention_kv8(const tidal_attn_kv8_args* a, void* d_ws, size_t ws_bytes, void* stream) {
    TIDAL_REQUIRE(a != nullptr, TIDAL_ERR_ARG, "args is NULL");
    TIDAL_REQUIRE(a->d_q && a->d_o && a->d_kv && a->d_scales, TIDAL_ERR_ARG, "attention_kv8: q, o, kv and scales must be given");
    TIDAL_REQUIRE((((uintptr_t)a->d_q | (uintptr_t)a->d_kv | (uintptr_t)a->d_o) & 15) == 0, TIDAL_ERR_ARG, "attention_kv8: q, o and kv must be 16-byte aligned");
    TIDAL_REQUIRE(a->batch >= 1 && a->num_qo_heads >= 1 && a->num_kv_heads >= 1, TIDAL_ERR_ARG, "attention_kv8: bad batch/heads");
    TIDAL_REQUIRE(a->num_qo_heads % a->num_kv_heads == 0, TIDAL_ERR_ARG, "num_qo_heads %d is not a multiple of num_kv_heads %d", a->num_qo_heads, a->num_kv_heads);
    TIDAL_REQUIRE(a->head_dim == 64 || a->head_dim == 128, TIDAL_ERR_ARG, "unsupported head_dim %d (built: 64, 128)", a->head_dim);
    TIDAL_REQUIRE(a->dtype >= 0 && a->dtype <= 2, TIDAL_ERR_ARG, "unknown dtype %d", a->dtype);
    TIDAL_REQUIRE(a->page_size >= 1 && a->num_pages >= 1, TIDAL_ERR_ARG, "bad page_size/num_pages");
    TIDAL_REQUIRE(a->block >= 1 && a->page_size % a->block == 0, TIDAL_ERR_ARG, "block %d does not divide page_size %d", a->block, a->page_size);
    TIDAL_REQUIRE(a->seq_len >= 0, TIDAL_ERR_ARG, "negative seq_len");
    TIDAL_REQUIRE(a->num_pages * 2 * a->page_size < ((int64_t)1 << 31), TIDAL_ERR_ARG, "the pool has 2^31 token rows or more (num_pages * 2 * page_size)");
    TIDAL_REQUIRE(a->num_pages * 2 * (a->page_size / a->block) * a->num_kv_heads < ((int64_t)1 << 32), TIDAL_ERR_ARG, "the pool has 2^32 scales or more");
    const bool sel = a->d_sel_idx != nullptr;
    if (sel) {
        TIDAL_REQUIRE(a->sel_rows == 1 || a->sel_rows == a->num_qo_heads, TIDAL_ERR_ARG, "sel_rows must be 1 or num_qo_heads, got %d", a->sel_rows);
        TIDAL_REQUIRE(a->sel_count >= 0 && a->sel_stride >= a->sel_count, TIDAL_ERR_ARG, "bad sel_count/sel_stride");
    }
    const int64_t pages = ((int64_t)a->seq_len + a->page_size - 1) / a->page_size;
    TIDAL_REQUIRE(!a->d_page_table || pages <= a->page_table_stride, TIDAL_ERR_ARG, "attention_kv8: the page table does not cover seq_len %d", a->seq_len);
    TIDAL_REQUIRE(a->d_page_table || (a->page_table_stride >= 0 && (int64_t)(a->batch - 1) * a->page_table_stride + pages <= a->num_pages), TIDAL_ERR_ARG,
                  "attention_kv8: identity page mapping runs past the pool's %lld pages", (long long)a->num_pages);
    const int ntok = sel ? a->sel_count : a->seq_len;
    TIDAL_REQUIRE(!a->d_scores || a->score_stride >= ntok, TIDAL_ERR_ARG, "score_stride shorter than the token list");
    const WsLayout* L = find_ws(d_ws);
    TIDAL_REQUIRE(L != nullptr, TIDAL_ERR_WORKSPACE, "workspace %p was not initialised with tidal_ws_init", d_ws);
    TIDAL_REQUIRE(ws_bytes >= L->total, TIDAL_ERR_WORKSPACE, "workspace is %zu bytes, layout needs %zu", ws_bytes, L->total);

    AttnKv8Params p;
    p.q = a->d_q; p.o = a->d_o; p.kv = (const uint8_t*)a->d_kv; p.scales = a->d_scales;
    p.map = SlotMap{a->d_page_table, a->page_table_stride, a->num_pages, a->page_size};
    p.seq_lens = a->d_seq_lens; p.seq_len = a->seq_len;
    p.sel_idx = a->d_sel_idx; p.sel_rows = sel ? a->sel_rows : 1; p.sel_count = a->sel_count; p.sel_stride = a->sel_stride;
    p.sel_counts = sel ? a->d_sel_counts : nullptr;
    p.scores = a->d_scores; p.score_stride = a->score_stride; p.lse = a->d_lse;
    p.part_o = (float*)((char*)d_ws + L->part_o_off);
    p.part_ml = (float*)((char*)d_ws + L->part_ml_off);
    p.status = (uint32_t*)((char*)d_ws + L->status_off);
    p.Hq = a->num_qo_heads; p.Hkv = a->num_kv_heads; p.G = a->num_qo_heads / a->num_kv_heads; p.block = a->block;
    p.sm_scale = a->sm_scale > 0.f ? a->sm_scale : 1.0f / sqrtf((float)a->head_dim);
    auto shift_of = [](int x) { return (x & (x - 1)) == 0 ? 31 - __builtin_clz((unsigned)x) : -1; };
    p.page_shift = shift_of(a->page_size);
    p.block_shift = shift_of(a->block);
    p.blocks_per_page = a->page_size / a->block;
    p.per_head = p.sel_rows != 1;
    const int64_t lists = (int64_t)a->batch * p.sel_rows;
    TIDAL_REQUIRE(lists <= 1 << 20, TIDAL_ERR_ARG, "attention_kv8: more than 2^20 token lists");
    p.lists = (int)lists;
    const int G = p.per_head ? 1 : p.G;
    p.groups = (G + 15) / 16;
    p.rows = (G + p.groups - 1) / p.groups;
    p.units = p.per_head ? 1 : p.Hkv * p.groups;
    p.ragged = sel ? p.sel_counts != nullptr : p.seq_lens != nullptr;
    p.pairs_per_list = ntok > 0 ? (ntok + 2 * kKv8Tile - 1) / (2 * kKv8Tile) : 1;
    const int64_t pairs = (int64_t)p.pairs_per_list * p.lists;
    TIDAL_REQUIRE(pairs <= INT32_MAX, TIDAL_ERR_ARG, "attention_kv8: more than 2^31 pairs of tiles");
    p.solo = ntok <= kKv8SoloTokens || p.lists > kKv8MaxPrefix;
    p.HC = 1;
    while (!p.solo && p.HC < 4 && p.units % (2 * p.HC) == 0) p.HC *= 2;
    p.slices = p.units / p.HC;
    const int TG = kKv8Warps / p.HC;
    if (p.solo) {
        p.ctas = p.lists;
    } else {
        // what is resident (two CTAs to an SM, or one, see attn_kv8_kernel), a pair at least to a warp, and no more parts than
        // the workspace holds
        const int per_sm = p.rows > 8 && (a->dtype == TIDAL_DTYPE_F32 || a->head_dim == 128) ? 1 : 2;
        int64_t ctas = std::max(1, per_sm * sm_count_cached() / p.slices);
        ctas = std::min(ctas, (pairs + TG - 1) / TG);
        const int64_t room = (int64_t)((L->part_ml_off - L->part_o_off) / (sizeof(float) * a->head_dim)) / ((int64_t)p.units * p.rows) - p.lists;
        ctas = std::min(ctas, room / TG);
        TIDAL_REQUIRE(ctas >= 1, TIDAL_ERR_WORKSPACE, "workspace was sized for a smaller batch/heads/head_dim than this call");
        p.ctas = (int)ctas;
    }
    p.ranges = p.ctas * TG;
    TIDAL_REQUIRE((int64_t)p.ctas * p.slices <= INT32_MAX, TIDAL_ERR_ARG, "attention_kv8: too many lists and heads");
    const size_t parts = (size_t)p.units * (p.ranges + p.lists) * p.rows;
    TIDAL_REQUIRE(p.solo || L->part_ml_off + sizeof(float) * parts * 2 <= L->hist_off, TIDAL_ERR_WORKSPACE,
                  "workspace was sized for a smaller batch/heads/head_dim than this call");
    cudaStream_t st = (cudaStream_t)stream;
    const bool wide = a->head_dim == 128;
    switch (a->dtype) {
        case TIDAL_DTYPE_F16: return wide ? launch_attn_kv8<__half, 128>(p, st) : launch_attn_kv8<__half, 64>(p, st);
        case TIDAL_DTYPE_BF16: return wide ? launch_attn_kv8<__nv_bfloat16, 128>(p, st) : launch_attn_kv8<__nv_bfloat16, 64>(p, st);
        default: return wide ? launch_attn_kv8<float, 128>(p, st) : launch_attn_kv8<float, 64>(p, st);
    }
}

TIDAL_TRACE_READER(tidal_trace_read_kv8)
