// Bounding a cache by what its tokens have been worth: softmax weights of a selection layer added up per token, and the
// pages of least weight moved out of a page table.
#include "common.cuh"

namespace tidal {

struct WeightsParams {
    const float* scores;
    int64_t score_stride;
    const float* lse;
    float* weights;
    int64_t weight_stride;
    const int32_t* seq_lens;
    int32_t seq_len, heads;
    float decay;
};

// w[j] = decay w[j] + sum_h exp(s[h][j] - lse[h]): one thread per token, heads in order.
__global__ void __launch_bounds__(256) accumulate_weights_kernel(const WeightsParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.y;
    const int len = p.seq_lens ? max(0, min(p.seq_lens[b], p.seq_len)) : p.seq_len;
    const int64_t j = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (j >= len) return;
    const float* s = p.scores + (size_t)b * p.heads * p.score_stride + j;
    float acc = 0.f;
    for (int h = 0; h < p.heads; ++h) {
        const float z = p.lse[(size_t)b * p.heads + h];
        const float w = fast_exp2((s[(size_t)h * p.score_stride] - z) * kLog2e);
        acc += z == -INFINITY ? 0.f : w;
    }
    float* w = p.weights + (size_t)b * p.weight_stride + j;
    *w = p.decay * *w + acc;
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
};

// Order-preserving key of a weight (see ordered_key); the two zeros are equal, every NaN is the greatest.
__device__ __forceinline__ uint32_t weight_key(float x) { return x != x ? 0xffffffffu : ordered_key(x + 0.f); }
// Key of page pg of a row of `len` tokens.
__device__ __forceinline__ uint32_t page_key(const float* w, int pg, int page_size, int len) {
    if (page_size == 1) return weight_key(w[pg]);
    const int t0 = pg * page_size, t1 = (int)min((int64_t)t0 + page_size, (int64_t)len);
    double sum = 0.0;
    for (int t = t0; t < t1; ++t) sum += (double)w[t];
    return weight_key((float)sum);
}

// Exclusive prefix over the CTA of a 0/1 flag per thread; *total receives the CTA's sum.  Every thread calls it.
__device__ __forceinline__ int block_rank(bool flag, int* total, int* warp_sums) {
    const uint32_t m = __ballot_sync(0xffffffffu, flag);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    __syncthreads();
    if (lane == 0) warp_sums[warp] = __popc(m);
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < warps; ++i) {
        const int c = warp_sums[i];
        before += i < warp ? c : 0;
        all += c;
    }
    *total = all;
    return before + __popc(m & ((1u << lane) - 1u));
}

// One CTA per row.  The keep - sink - recent heaviest of the pages between the protected ones are found by a radix
// select over their keys, four digits of eight bits from the top; equal keys at the threshold go to the lower pages.
// Then one walk over the pages in order gives every page its place.
__global__ void __launch_bounds__(1024) evict_pages_kernel(const EvictParams p) {
    __shared__ uint32_t hist[256];
    __shared__ int warp_sums[32];
    __shared__ uint32_t s_digit;
    __shared__ int s_need;
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.x;
    const float* w = p.weights + (size_t)row * p.weight_stride;
    float* w_out = p.weights_out + (size_t)row * p.weight_stride;
    const int32_t* table = p.table + (size_t)row * p.table_stride;
    int32_t* table_out = p.table_out + (size_t)row * p.table_stride;
    const int len = p.seq_lens ? max(0, min(p.seq_lens[row], p.max_len)) : p.max_len;
    const int used = (int)(((int64_t)len + p.page_size - 1) / p.page_size);
    const int max_pages = (int)(((int64_t)p.max_len + p.page_size - 1) / p.page_size);
    const int tid = threadIdx.x, nt = blockDim.x;
    if (used <= p.keep) {
        for (int i = tid; i < max_pages; i += nt) table_out[i] = table[i];
        for (int i = tid; i < p.max_len; i += nt) w_out[i] = w[i];
        if (tid == 0) p.seq_lens_out[row] = len;
        return;
    }
    const int lo = p.sink, hi = used - p.recent;                 // the pages that compete
    int need = p.keep - p.sink - p.recent;                       // of them stay
    uint32_t prefix = 0;                                         // the threshold key, digit by digit
    if (need > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += nt) hist[i] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += nt) {
                const uint32_t k = page_key(w, i, p.page_size, len);
                if (shift == 24 || k >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist[k >> shift & 255u], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                int left = need, d = 255;
                while (d > 0 && (int)hist[d] < left) left -= (int)hist[d--];
                s_digit = (uint32_t)d;
                s_need = left;
            }
            __syncthreads();
            prefix |= s_digit << shift;
            need = s_need;                                       // how many with exactly these leading digits stay
        }
    }
    int kept = 0, gone = 0, ties = 0;
    for (int i0 = 0; i0 < used; i0 += nt) {
        const int i = i0 + tid;
        const bool in = i < used;
        const bool competes = in && i >= lo && i < hi;
        const uint32_t k = competes ? page_key(w, i, p.page_size, len) : 0u;
        const bool any = p.keep > p.sink + p.recent;
        const bool tie = competes && any && k == prefix;
        int total;
        const int tie_rank = ties + block_rank(tie, &total, warp_sums);
        ties += total;
        const bool stay = in && (!competes || (any && (k > prefix || (tie && tie_rank < need))));
        const int r = kept + block_rank(stay, &total, warp_sums);
        kept += total;
        const int g = gone + block_rank(in && !stay, &total, warp_sums);
        gone += total;
        if (in) table_out[stay ? r : p.keep + g] = table[i];
        if (stay) {
            const int t0 = i * p.page_size, t1 = (int)min((int64_t)t0 + p.page_size, (int64_t)len);
            for (int t = t0; t < t1; ++t) w_out[r * p.page_size + (t - t0)] = w[t];
        }
    }
    const int new_len = len - (used - p.keep) * p.page_size;
    for (int i = used + tid; i < max_pages; i += nt) table_out[i] = table[i];
    for (int i = new_len + tid; i < len; i += nt) w_out[i] = 0.f;
    for (int i = len + tid; i < p.max_len; i += nt) w_out[i] = w[i];
    if (tid == 0) p.seq_lens_out[row] = new_len;
}

}  // namespace tidal

using namespace tidal;

extern "C" int tidal_accumulate_weights(const tidal_weights_args* a, void* stream) {
    TIDAL_REQUIRE(a != nullptr, TIDAL_ERR_ARG, "args is NULL");
    TIDAL_REQUIRE(a->d_scores && a->d_lse && a->d_weights, TIDAL_ERR_ARG, "accumulate_weights: scores, lse and weights must be given");
    TIDAL_REQUIRE(a->batch >= 1 && a->batch <= 65535 && a->heads >= 1, TIDAL_ERR_ARG, "accumulate_weights: bad batch/heads");
    TIDAL_REQUIRE(a->seq_len >= 0 && a->score_stride >= a->seq_len && a->weight_stride >= a->seq_len, TIDAL_ERR_ARG,
                  "accumulate_weights: rows of scores or weights shorter than seq_len %d", a->seq_len);
    if (a->seq_len == 0) return TIDAL_OK;
    WeightsParams p{a->d_scores, a->score_stride, a->d_lse, a->d_weights, a->weight_stride, a->d_seq_lens, a->seq_len, a->heads, a->decay};
    TIDAL_CUDA_OK(launch_pdl(accumulate_weights_kernel, dim3((unsigned)((a->seq_len + 255LL) / 256), a->batch), dim3(256), 0, (cudaStream_t)stream, 1, p));
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
                  a->d_seq_lens, a->d_seq_lens_out, a->max_len, a->page_size, a->keep_pages, a->sink_pages, a->recent_pages};
    TIDAL_CUDA_OK(launch_pdl(evict_pages_kernel, dim3(a->rows), dim3(1024), 0, (cudaStream_t)stream, 1, p));
    count_launch();
    return TIDAL_OK;
}
