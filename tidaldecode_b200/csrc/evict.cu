// Bounding a cache by what its tokens have been worth: softmax weights of a selection layer added up per token, and the
// pages of least weight moved out of a page table.
#include <algorithm>
#include <type_traits>

#include <cooperative_groups.h>

#include "common.cuh"

namespace tidal {

struct WeightsParams {
    const float* scores;
    int64_t score_stride;
    const float* lse;
    float* weights;
    int64_t weight_stride;
    const int32_t* seq_lens;
    int32_t seq_len, heads, batch, strips, warps;     // strips of seq_len tokens; warps that fill the device
    float decay;
};

// Inclusive prefix over the CTA's threads; `sums` holds one word per warp.  Every thread calls it.
__device__ __forceinline__ int block_inclusive(int x, int* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    int s = lane < (int)(blockDim.x >> 5) ? sums[lane] : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, s, off);
        if (lane >= off) s += y;
    }
    return x + (warp > 0 ? __shfl_sync(0xffffffffu, s, warp - 1) : 0);
}

// w[j] = decay w[j] + sum_h exp(s[h][j] - lse[h]).  A warp takes 128 tokens of every HW-th head, four tokens to a lane (one
// 16-byte load where rows allow it) and eight heads in flight; the HW warps' sums meet in shared memory in the order of
// the warps, so the result does not depend on timing.  A few CTAs per SM walk over the strips of all sequences end to end
// (every CTA adds the lengths up itself): with a grid over the longest possible sequence most CTAs of a ragged batch had
// nothing to do (17.8 us instead of 11.4 for 8 sequences of up to 128 K tokens, 36 MB).  Bound by HBM / L2: the logits are read
// once; 8 full sequences of 128 K tokens x 32 heads, 136 MB: 25 us, 5.3 TB/s.
constexpr int kWeightTokens = 128;
constexpr int kWeightBatch = 1024;       // sequences whose lengths a CTA adds up
template <bool VEC>
__global__ void __launch_bounds__(256, 4) accumulate_weights_kernel(const WeightsParams p) {
    __shared__ float sums[8][kWeightTokens];
    __shared__ int before[kWeightBatch + 1], scan[32];           // steps before each sequence
    pdl_wait();
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto strips_of = [&](int i) -> int {
        const int n = i < p.batch ? min(p.seq_lens[i], p.seq_len) : 0;
        return n > 0 ? (n - 1) / kWeightTokens + 1 : 0;
    };
    int64_t total;                                               // strips of all sequences
    if (p.seq_lens) {
        int own = 0;
        const int first = threadIdx.x * (kWeightBatch / 256);
        for (int i = 0; i < kWeightBatch / 256; ++i) own += strips_of(first + i);
        int at = block_inclusive(own, scan) - own;
        for (int i = 0; i < kWeightBatch / 256; ++i) {
            before[first + i] = at;
            at += strips_of(first + i);
        }
        if (threadIdx.x == 255) before[kWeightBatch] = at;
        __syncthreads();
        total = before[kWeightBatch];
    } else {
        total = (int64_t)p.batch * p.strips;
    }
    // warps per strip: as many as heads (up to 8) while there are few strips, one (no barrier) when the strips alone fill the
    // SMs (8 sequences of 128 K tokens, 32 heads: 40 us with 8 warps to a strip, 25 with one)
    int hw = p.heads >= 8 ? 8 : p.heads >= 4 ? 4 : p.heads >= 2 ? 2 : 1;
    while (hw > 1 && total * hw > p.warps) hw >>= 1;
    const int per_cta = 8 / hw, h0 = warp % hw;
    for (int64_t step = blockIdx.x; step * per_cta < total; step += gridDim.x) {
        const int64_t q = step * per_cta + warp / hw;            // this warp's strip
        int b = 0, strip = 0;
        if (p.seq_lens) {
            int hi = kWeightBatch;                               // last sequence that starts at or before the strip
            while (hi - b > 1) {
                const int mid = (b + hi) >> 1;
                if (before[mid] <= q) b = mid; else hi = mid;
            }
            strip = (int)(q - before[b]);
        } else if (q < total) {
            b = (int)(q / p.strips);
            strip = (int)(q - (int64_t)b * p.strips);
        }
        const int len = q >= total ? 0 : p.seq_lens ? min(p.seq_lens[b], p.seq_len) : p.seq_len;
        if (q >= total) b = 0, strip = 0;
        const int64_t j0 = (int64_t)strip * kWeightTokens;       // token of lane 0
        const float* s = p.scores + (size_t)b * p.heads * p.score_stride + j0;
        const float* z = p.lse + (size_t)b * p.heads;
        float acc[4] = {};
        auto add = [&](const float (&x)[4], float zh) {
            if (zh == -INFINITY) return;                         // a row without tokens adds nothing
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += fast_exp2((x[i] - zh) * kLog2e);
        };
        const size_t stride = (size_t)hw * p.score_stride;
        const float* row = s + (size_t)h0 * p.score_stride;
        if (VEC && j0 + kWeightTokens <= len) {
            const float* at = row + 4 * lane;
            int h = h0;
            auto batch = [&](auto count) {                       // as many heads as their loads are in flight together
                constexpr int K = decltype(count)::value;
                for (; h + (K - 1) * hw < p.heads; h += K * hw, at += K * stride) {
                    float4 v[K];
                    float zh[K];
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        v[k] = __ldcs(reinterpret_cast<const float4*>(at + k * stride));
                        zh[k] = z[h + k * hw];
                    }
#pragma unroll
                    for (int k = 0; k < K; ++k) add({v[k].x, v[k].y, v[k].z, v[k].w}, zh[k]);
                }
            };
            batch(std::integral_constant<int, 8>());
            batch(std::integral_constant<int, 4>());
            batch(std::integral_constant<int, 1>());
        } else if (j0 < len) {
            for (int h = h0; h < p.heads; h += hw, row += stride) {
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = VEC ? 4 * lane + i : lane + 32 * i;
                    x[i] = j0 + t < len ? row[t] : 0.f;
                }
                add(x, z[h]);
            }
        }
        float* w = p.weights + (size_t)b * p.weight_stride + j0;
        if (hw == 1) {                                           // the warp has its tokens' sums: no other warp is waited for
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = VEC ? 4 * lane + i : lane + 32 * i;
                if (j0 + t < len) w[t] = p.decay * w[t] + acc[i];
            }
            continue;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[warp][VEC ? 4 * lane + i : lane + 32 * i] = acc[i];
        __syncthreads();
        for (int t = h0 * 32 + lane; t < kWeightTokens && j0 + t < len; t += 32 * hw) {
            float sum = 0.f;
            for (int k = 0; k < hw; ++k) sum += sums[warp - h0 + k][t];
            w[t] = p.decay * w[t] + sum;
        }
        __syncthreads();
    }
}

struct EvictParams {
    const float* weights;
    float* weights_out;
    int64_t weight_stride;
    const int32_t* table;
    int32_t* table_out;
    int64_t table_stride;
    const int32_t* seq_lens;
    int32_t* seq_lens_out;
    int32_t max_len, page_size, keep, sink, recent;
    int32_t cached;              // page keys are kept in shared memory
    int32_t row_vec4, table_vec4;// rows of weights / of the table start on 16 bytes
    int32_t vec4;                // ... and so do the pages of weights
    int32_t page_shift;          // of page_size, or of page_size / 4 with vec4; -1: no power of two
};

// Order-preserving key of a weight (see ordered_key); the two zeros are equal, every NaN is the greatest.
__device__ __forceinline__ uint32_t weight_key(float x) { return x != x ? 0xffffffffu : ordered_key(x + 0.f); }
// Key of page pg of a row of `len` tokens.
__device__ __forceinline__ uint32_t page_key(const float* w, int pg, int page_size, int len, bool vec4) {
    if (page_size == 1) return weight_key(w[pg]);
    const int t0 = pg * page_size, t1 = (int)min((int64_t)t0 + page_size, (int64_t)len);
    double sum = 0.0;
    int t = t0;
    if (vec4)
        for (; t + 4 <= t1; t += 4) {
            const float4 v = *reinterpret_cast<const float4*>(w + t);
            sum += ((double)v.x + (double)v.y) + ((double)v.z + (double)v.w);
        }
    for (; t < t1; ++t) sum += (double)w[t];
    return weight_key((float)sum);
}

// dst[i] = src[i] (src NULL: 0) for from <= i < to, by threads me of `all`; vec4: dst and src start on 16 bytes, and the
// vectors that lie in the range whole go as such.  Out of line: it is called in several places of a kernel whose
// instructions are fetched cold.
static __device__ __noinline__ void copy_row(uint32_t* dst, const uint32_t* src, uint32_t from, uint32_t to, uint32_t me, uint32_t all, bool vec4) {
    if (vec4) {
        const uint32_t a = min((from + 3) / 4, (to + 3) / 4), b = max(to / 4, a);
        if (me < a * 4 - from && from + me < to) dst[from + me] = src ? src[from + me] : 0u;
#pragma unroll 4
        for (uint32_t v = a + me; v < b; v += all) reinterpret_cast<uint4*>(dst)[v] = src ? reinterpret_cast<const uint4*>(src)[v] : make_uint4(0, 0, 0, 0);
        from = max(b * 4, from);
    }
    for (uint32_t k = from + me; k < to; k += all) dst[k] = src ? src[k] : 0u;
}

constexpr int kEvictThreads = 1024;
constexpr int kEvictBins = 2048;          // 11-bit digits, from the top: 11 + 11 + 10 bits
constexpr int kEvictFew = 256;            // keys that are ranked by comparing each with each
constexpr int kEvictKeys = 47 * 1024;     // page keys a CTA keeps in shared memory; beyond that they are formed anew

// A cluster per row, each of its CTAs with a contiguous part of the row's pages.  The keep - sink - recent heaviest of the
// pages between the protected ones are found by a radix select over their keys: a histogram per CTA and digit, added up
// through distributed shared memory by every CTA, so that all know the threshold after one cluster barrier per digit.
// Equal keys at the threshold go to the lower pages.  A warp owns 32-page groups in order; two walks over them (count,
// then place) with one prefix over the warps and one over the CTAs between them give every page its place.
// Bound by latency: one to three histogram passes, up to four cluster barriers; the bytes are nothing beside them.  One row of
// 4096 single-token pages 9.6 us (31.6 with one CTA that formed the keys anew in every pass), 32 rows of up to 128 K tokens
// in pages of 16: 20 us (266).
__global__ void __launch_bounds__(kEvictThreads) evict_pages_kernel(const EvictParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ uint32_t keys[];
    __shared__ uint2 hist2[3][kEvictBins / 2];                   // read in pairs: by type on 8 bytes
    __shared__ uint32_t few[kEvictFew];
    __shared__ int sums[32], s_pick[3], s_ties, s_more, s_few;
    __shared__ int warp_ties[32], warp_more[32];
    uint32_t (*const hist)[kEvictBins] = reinterpret_cast<uint32_t (*)[kEvictBins]>(hist2);
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i < 3 * kEvictBins; i += kEvictThreads) (&hist[0][0])[i] = 0;
    if (tid == 0) s_few = 0;
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.x / C;
    const float* w = p.weights + (size_t)row * p.weight_stride;
    float* w_out = p.weights_out + (size_t)row * p.weight_stride;
    const int32_t* table = p.table + (size_t)row * p.table_stride;
    int32_t* table_out = p.table_out + (size_t)row * p.table_stride;
    const int len = p.seq_lens ? max(0, min(p.seq_lens[row], p.max_len)) : p.max_len;
    const int ps = p.page_size;
    const int used = (int)(((int64_t)len + ps - 1) / ps);
    const int max_pages = (int)(((int64_t)p.max_len + ps - 1) / ps);
    const uint32_t me = (uint32_t)(rank * kEvictThreads + tid), all = (uint32_t)(C * kEvictThreads);
    if (used <= p.keep) {                                        // the whole cluster agrees
        copy_row((uint32_t*)table_out, (const uint32_t*)table, 0, max_pages, me, all, p.table_vec4 != 0);
        copy_row((uint32_t*)w_out, (const uint32_t*)w, 0, p.max_len, me, all, p.row_vec4 != 0);
        if (me == 0) p.seq_lens_out[row] = len;
        return;
    }
    const int new_len = len - (used - p.keep) * ps;
    copy_row((uint32_t*)table_out, (const uint32_t*)table, used, max_pages, me, all, p.table_vec4 != 0);
    copy_row((uint32_t*)w_out, nullptr, new_len, len, me, all, p.row_vec4 != 0);
    copy_row((uint32_t*)w_out, (const uint32_t*)w, len, p.max_len, me, all, p.row_vec4 != 0);
    if (me == 0) p.seq_lens_out[row] = new_len;

    // ---- this CTA's pages [base, base + n), and of each warp the 32-page groups [g0, g1) of them
    const int groups = (used + 31) / 32, per_cta = (groups + C - 1) / C;
    const int base = min(rank * per_cta, groups) * 32, n = min(used - base, per_cta * 32);
    const int mine = n > 0 ? (n + 31) / 32 : 0, per_warp = (mine + 31) / 32;
    const int g0 = min(warp * per_warp, mine), g1 = min(g0 + per_warp, mine);
    const int lo = p.sink, hi = used - p.recent;                 // the pages that compete
    const int places = p.keep - p.sink - p.recent;               // of them stay
    const bool cached = p.cached != 0;
    const bool vec4 = p.vec4 != 0;
    auto key_of = [&](int i) -> uint32_t { return cached ? keys[i] : page_key(w, base + i, ps, len, vec4); };
    if (cached)
#pragma unroll 4
        for (int i = tid; i < n; i += kEvictThreads) keys[i] = page_key(w, base + i, ps, len, vec4);
    __syncthreads();

    uint32_t threshold = 0;
    int need = places;                                           // how many of the keys with the threshold's leading digits stay
    if (places > 0) {
        bool found = false;
#pragma unroll
        for (int d = 0; d < 3 && !found; ++d) {
            const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, bits = d == 2 ? 10 : 11;
            for (int i = tid; i < n; i += kEvictThreads) {
                const int pg = base + i;
                const uint32_t k = key_of(i);
                if (pg >= lo && pg < hi && (d == 0 || k >> (shift + bits) == threshold >> (shift + bits)))
                    atomicAdd(&hist[d][k >> shift & ((1u << bits) - 1u)], 1u);
            }
            if (C > 1) cluster.sync();
            else __syncthreads();
            // thread t takes the bins 2047 - 2t and 2046 - 2t: a prefix over the threads counts from the greatest key down
            const int bin = kEvictBins - 2 - 2 * tid;
            int c0 = 0, c1 = 0;
            for (int r = 0; r < C; ++r) {
                const uint2 v = (C > 1 ? cluster.map_shared_rank(&hist2[d][0], r) : &hist2[d][0])[bin / 2];
                c0 += (int)v.x;
                c1 += (int)v.y;
            }
            const int upto = block_inclusive(c0 + c1, sums), before = upto - c0 - c1;
            if (before < need && need <= upto) {                 // exactly one thread: there are at least `need` such keys
                const bool high = need <= before + c1;
                s_pick[0] = bin + (high ? 1 : 0);
                s_pick[1] = need - before - (high ? 0 : c1);
                s_pick[2] = high ? c1 : c0;                      // keys with these leading digits
            }
            __syncthreads();
            threshold |= (uint32_t)s_pick[0] << shift;
            need = s_pick[1];
            if (d == 0 && C == 1 && s_pick[2] <= kEvictFew) {
                // few keys share the first digit, as a rule: they are ranked against each other, in place of two more histograms
                // (across CTAs the gathering cost more than it saved: 26 us instead of 20 for 8192 pages)
                for (int i = tid; i < n; i += kEvictThreads) {
                    const int pg = base + i;
                    const uint32_t k = key_of(i);
                    if (pg >= lo && pg < hi && k >> shift == threshold >> shift) few[atomicAdd(&s_few, 1)] = k;
                }
                __syncthreads();
                const int count = s_few;
                if (tid < count) {
                    const uint32_t k = few[tid];
                    int above = 0, same = 0;
#pragma unroll 4
                    for (int i = 0; i < count; ++i) {
                        above += few[i] > k ? 1 : 0;
                        same += few[i] == k ? 1 : 0;
                    }
                    if (above < need && need <= above + same) {  // the same for every key equal to the threshold
                        s_pick[0] = (int)k;
                        s_pick[1] = need - above;
                    }
                }
                __syncthreads();
                threshold = (uint32_t)s_pick[0];
                need = s_pick[1];
                found = true;
            }
        }
    }

    // ---- first walk: how many of each warp's pages lie above the threshold (or are protected), how many at it
    auto classify = [&](int gr, bool* in, bool* tie) -> bool {
        const int i = gr * 32 + lane, pg = base + i;
        *in = i < n;
        const bool competes = *in && pg >= lo && pg < hi;
        const uint32_t k = competes ? key_of(i) : 0u;
        *tie = competes && places > 0 && k == threshold;
        return *in && (!competes || (places > 0 && k > threshold));
    };
    int ties = 0, more = 0;
    for (int gr = g0; gr < g1; ++gr) {
        bool in, tie;
        const bool above = classify(gr, &in, &tie);
        more += __popc(__ballot_sync(0xffffffffu, above));
        ties += __popc(__ballot_sync(0xffffffffu, tie));
    }
    if (lane == 0) warp_ties[warp] = ties, warp_more[warp] = more;
    __syncthreads();
    if (warp == 0) {
        int a = warp_ties[lane], b = warp_more[lane];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, a, off), z = __shfl_up_sync(0xffffffffu, b, off);
            if (lane >= off) a += y, b += z;
        }
        if (lane == 31) s_ties = a, s_more = b;
        const int ta = __shfl_up_sync(0xffffffffu, a, 1), tb = __shfl_up_sync(0xffffffffu, b, 1);
        warp_ties[lane] = lane > 0 ? ta : 0;
        warp_more[lane] = lane > 0 ? tb : 0;
    }
    if (C > 1) cluster.sync();
    else __syncthreads();
    int tie_at = warp_ties[warp], more_at = warp_more[warp];     // ties and sure pages before this warp's
    for (int r = 0; r < rank; ++r) {
        tie_at += *cluster.map_shared_rank(&s_ties, r);
        more_at += *cluster.map_shared_rank(&s_more, r);
    }
    if (C > 1) cluster_arrive_release();                         // done with the other CTAs' shared memory; waited for before leaving

    // ---- second walk: every page to its place
    const uint32_t below = (1u << lane) - 1u;
    constexpr int kAhead = 4;                                    // groups whose table entries and weights are loaded together
    for (int gr0 = g0; gr0 < g1; gr0 += kAhead) {
        int32_t entry[kAhead];
        float weight[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = (gr0 + k) * 32 + lane;
            const bool in = gr0 + k < g1 && i < n;
            entry[k] = in ? table[base + i] : 0;
            weight[k] = in && ps == 1 ? w[base + i] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int gr = gr0 + k;
            if (gr >= g1) break;
            bool in, tie;
            const bool above = classify(gr, &in, &tie);
            const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie), sure_mask = __ballot_sync(0xffffffffu, above);
            const bool stay = above || (tie && tie_at + __popc(tie_mask & below) < need);
            const uint32_t stay_mask = __ballot_sync(0xffffffffu, stay);
            const int i = base + gr * 32 + lane;
            const int r = more_at + min(tie_at, need) + __popc(stay_mask & below);  // kept pages before this one
            if (in) table_out[stay ? r : p.keep + i - r] = entry[k];
            if (ps == 1) {
                if (stay) w_out[r] = weight[k];
            } else {
                // the group's 32 pages end to end, four (or one) weights to a lane: independent loads, whatever the page size
                const int first = (base + gr * 32) * ps, width = vec4 ? 4 : 1, steps = ps / width;
#pragma unroll 4
                for (int e = lane; e < 32 * steps; e += 32) {
                    const int src = p.page_shift >= 0 ? e >> p.page_shift : e / steps, at = (e - src * steps) * width;
                    const int to = __shfl_sync(0xffffffffu, r, src) * ps + at, from = first + src * ps + at;
                    if (!(stay_mask >> src & 1u)) continue;
                    if (width == 4 && from + 4 <= len) *reinterpret_cast<float4*>(w_out + to) = *reinterpret_cast<const float4*>(w + from);
                    else
                        for (int j = 0; j < width; ++j)
                            if (from + j < len) w_out[to + j] = w[from + j];
                }
            }
            tie_at += __popc(tie_mask);
            more_at += __popc(sure_mask);
        }
    }
    if (C > 1) cluster_wait();
}

}  // namespace tidal

using namespace tidal;

extern "C" int tidal_accumulate_weights(const tidal_weights_args* a, void* stream) {
    TIDAL_REQUIRE(a != nullptr, TIDAL_ERR_ARG, "args is NULL");
    TIDAL_REQUIRE(a->d_scores && a->d_lse && a->d_weights, TIDAL_ERR_ARG, "accumulate_weights: scores, lse and weights must be given");
    TIDAL_REQUIRE(a->batch >= 1 && (!a->d_seq_lens || a->batch <= kWeightBatch) && a->heads >= 1, TIDAL_ERR_ARG, "accumulate_weights: bad heads or batch (%d; at most %d sequences of different lengths)", a->batch, kWeightBatch);
    TIDAL_REQUIRE(a->seq_len >= 0 && a->score_stride >= a->seq_len && a->weight_stride >= a->seq_len, TIDAL_ERR_ARG,
                  "accumulate_weights: rows of scores or weights shorter than seq_len %d", a->seq_len);
    if (a->seq_len == 0) return TIDAL_OK;
    const int strips = (int)((a->seq_len + (int64_t)kWeightTokens - 1) / kWeightTokens);
    const WeightsParams p{a->d_scores, a->score_stride, a->d_lse, a->d_weights, a->weight_stride, a->d_seq_lens, a->seq_len, a->heads, a->batch, strips,
                          40 * sm_count_cached(), a->decay};
    const dim3 grid((unsigned)std::min<int64_t>((int64_t)a->batch * strips, 4 * sm_count_cached()));
    const bool vec = a->score_stride % 4 == 0 && ((uintptr_t)a->d_scores & 15) == 0;
    if (vec) TIDAL_CUDA_OK(launch_pdl(accumulate_weights_kernel<true>, grid, dim3(256), 0, (cudaStream_t)stream, 1, p));
    else TIDAL_CUDA_OK(launch_pdl(accumulate_weights_kernel<false>, grid, dim3(256), 0, (cudaStream_t)stream, 1, p));
    count_launch();
    return TIDAL_OK;
}

extern "C" int tidal_evict_pages(const tidal_evict_args* a, void* stream) {
    TIDAL_REQUIRE(a != nullptr, TIDAL_ERR_ARG, "args is NULL");
    TIDAL_REQUIRE(a->d_weights && a->d_weights_out && a->d_page_table && a->d_page_table_out && a->d_seq_lens_out, TIDAL_ERR_ARG,
                  "evict_pages: weights, page_table, seq_lens and their outputs must be given");
    TIDAL_REQUIRE(a->rows >= 1 && a->page_size >= 1 && a->max_len >= 1, TIDAL_ERR_ARG, "evict_pages: bad rows/page_size/max_len");
    TIDAL_REQUIRE(a->sink_pages >= 0 && a->recent_pages >= 1, TIDAL_ERR_ARG,
                  "evict_pages: sink_pages must be >= 0 and recent_pages >= 1 (the last page may be partly filled)");
    TIDAL_REQUIRE((int64_t)a->sink_pages + a->recent_pages <= a->keep_pages, TIDAL_ERR_ARG, "evict_pages: keep_pages %d is less than sink_pages %d + recent_pages %d",
                  a->keep_pages, a->sink_pages, a->recent_pages);
    const int64_t max_pages = ((int64_t)a->max_len + a->page_size - 1) / a->page_size;
    TIDAL_REQUIRE(a->weight_stride >= a->max_len && a->page_table_stride >= max_pages, TIDAL_ERR_ARG,
                  "evict_pages: rows of weights or page_table shorter than max_len %d", a->max_len);
    const char *w = (const char*)a->d_weights, *wo = (const char*)a->d_weights_out, *t = (const char*)a->d_page_table, *to = (const char*)a->d_page_table_out;
    const size_t wb = sizeof(float) * ((size_t)(a->rows - 1) * a->weight_stride + a->max_len);
    const size_t tb = sizeof(int32_t) * ((size_t)(a->rows - 1) * a->page_table_stride + max_pages);
    const char *l = (const char*)a->d_seq_lens, *lo = (const char*)a->d_seq_lens_out;
    const size_t lb = sizeof(int32_t) * (size_t)a->rows;
    TIDAL_REQUIRE((w + wb <= wo || wo + wb <= w) && (t + tb <= to || to + tb <= t) && (!l || l + lb <= lo || lo + lb <= l), TIDAL_ERR_ARG,
                  "evict_pages: outputs overlap the inputs");
    EvictParams p{a->d_weights, a->d_weights_out, a->weight_stride, a->d_page_table, a->d_page_table_out, a->page_table_stride,
                  a->d_seq_lens, a->d_seq_lens_out, a->max_len, a->page_size, a->keep_pages, a->sink_pages, a->recent_pages, 0, 0, 0, 0, -1};
    p.row_vec4 = a->weight_stride % 4 == 0 && (((uintptr_t)a->d_weights | (uintptr_t)a->d_weights_out) & 15) == 0;
    p.table_vec4 = a->page_table_stride % 4 == 0 && (((uintptr_t)a->d_page_table | (uintptr_t)a->d_page_table_out) & 15) == 0;
    p.vec4 = p.row_vec4 && a->page_size % 4 == 0;
    const int steps = p.vec4 ? a->page_size / 4 : a->page_size;
    if ((steps & (steps - 1)) == 0) p.page_shift = 31 - __builtin_clz((unsigned)steps);
    // CTAs per row: one CTA takes 1.3 us for every 1024 pages and as much for 4096 weights of longer pages; a second, the
    // fourth and the eighth each add 2 us or more of barriers.  Measured, in us, with 1 / 2 / 4 / 8 CTAs: 4096 single-token
    // pages 9.6 / 10.8 / 11.7 / 14.5, 16 K 22.5 / 16.7 / 14.5 / 16.5, 128 K 177 / 96 / 43 / 31, 8192 pages of 16 tokens
    // 37 / 25 / 19 / 20.  Clusters beyond one to an SM would wait for each other (32 rows of 32 K: 19 with 4, 55 with 8).
    const int64_t load = max_pages + (a->page_size > 1 ? a->max_len / 4 : 0);
    int C = load < 6144 ? 1 : load < 12288 ? 2 : load < 45056 ? 4 : 8;
    while (C > 1 && (int64_t)a->rows * C > sm_count_cached()) C /= 2;
    TIDAL_REQUIRE((int64_t)a->rows * C <= INT32_MAX, TIDAL_ERR_ARG, "evict_pages: too many rows");
    const int64_t per_cta = ((max_pages + 31) / 32 + C - 1) / C * 32;
    const size_t smem = sizeof(uint32_t) * (size_t)(per_cta <= kEvictKeys ? per_cta : 0);
    p.cached = smem > 0;
    if (smem > 16384) TIDAL_CUDA_OK(cudaFuncSetAttribute(evict_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvictKeys * 4));
    TIDAL_CUDA_OK(launch_pdl(evict_pages_kernel, dim3(a->rows * C), dim3(kEvictThreads), smem, (cudaStream_t)stream, C, p));
    count_launch();
    return TIDAL_OK;
}
