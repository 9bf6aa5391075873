// One decode step of attention over an 8-bit KV pool.
#include "kv8.cuh"

namespace tidal {

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
    float* part_o;               // [B * Hq][chunks][D]
    float* part_ml;              // [B * Hq][chunks][2]
    uint32_t* status;
    int32_t Hq, Hkv, G, block, chunks;
    float sm_scale;
};

constexpr int kKv8Warps = 4;

// One CTA per (query head, chunk of its token list); a warp takes every fourth token, its lanes the elements.
template <typename T, int D>
__global__ void __launch_bounds__(kKv8Warps * 32) attn_kv8_kernel(const AttnKv8Params p) {
    constexpr int EPL = D / 32;
    __shared__ float sh_o[kKv8Warps][D];
    __shared__ float sh_ml[kKv8Warps][2];
    pdl_wait();
    pdl_launch_dependents();
    const int chunk = blockIdx.x, hq = blockIdx.y % p.Hq, b = blockIdx.y / p.Hq;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = hq / p.G;
    const int seq = p.seq_lens ? max(0, min(p.seq_lens[b], p.seq_len)) : p.seq_len;
    const size_t list = p.sel_rows == 1 ? b : (size_t)b * p.Hq + hq;
    int n = seq;
    if (p.sel_idx) n = p.sel_counts ? max(0, min(p.sel_counts[list], p.sel_count)) : p.sel_count;
    const int per = (n + p.chunks - 1) / p.chunks;
    const int t0 = chunk * per, t1 = min(n, t0 + per);
    float q[EPL];
    const T* qrow = reinterpret_cast<const T*>(p.q) + ((size_t)b * p.Hq + hq) * D + lane * EPL;
#pragma unroll
    for (int i = 0; i < EPL; ++i) q[i] = to_f32(qrow[i]);
    float m = -INFINITY, l = 0.f, o[EPL] = {};
    for (int t = t0 + warp; t < t1; t += kKv8Warps) {
        const int pos = p.sel_idx ? p.sel_idx[list * p.sel_stride + t] : t;
        int entry = 0;
        int64_t page = pos >= seq ? -1 : p.map.page_of(b, pos, &entry);
        if (page < 0) {
            if (lane == 0) atomicOr(p.status, TIDAL_DEV_BAD_INDEX);
            continue;
        }
        const int ps = p.map.page_size;
        float kv[2][EPL];
#pragma unroll
        for (int pl = 0; pl < 2; ++pl) {
            const uint8_t* c = p.kv + (((size_t)page * 2 + pl) * ps + entry) * p.Hkv * D + (size_t)h * D + lane * EPL;
            const float sc = scale_value(p.scales[(((size_t)page * 2 + pl) * (ps / p.block) + entry / p.block) * p.Hkv + h]);
#pragma unroll
            for (int i = 0; i < EPL; i += 2) {
                const float2 f = unpack_e4m3(*reinterpret_cast<const uint16_t*>(c + i));
                kv[pl][i] = f.x * sc;
                kv[pl][i + 1] = f.y * sc;
            }
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < EPL; ++i) s += q[i] * kv[0][i];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        s *= p.sm_scale;
        if (p.scores && lane == 0) p.scores[((size_t)b * p.Hq + hq) * p.score_stride + t] = s;
        s *= kLog2e;
        const float mn = fmaxf(m, s), keep = mn == -INFINITY ? 1.f : fast_exp2(m - mn), w = mn == -INFINITY ? 0.f : fast_exp2(s - mn);
        m = mn;
        l = l * keep + w;
#pragma unroll
        for (int i = 0; i < EPL; ++i) o[i] = o[i] * keep + w * kv[1][i];
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) sh_o[warp][lane * EPL + i] = o[i];
    if (lane == 0) sh_ml[warp][0] = m, sh_ml[warp][1] = l;
    __syncthreads();
    const size_t part = ((size_t)b * p.Hq + hq) * p.chunks + chunk;
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
        float M = -INFINITY, L = 0.f, acc = 0.f;
        for (int i = 0; i < kKv8Warps; ++i) M = fmaxf(M, sh_ml[i][0]);
        for (int i = 0; i < kKv8Warps; ++i) {
            const float w = sh_ml[i][0] == -INFINITY ? 0.f : fast_exp2(sh_ml[i][0] - M);
            L += w * sh_ml[i][1];
            acc += w * sh_o[i][d];
        }
        p.part_o[part * D + d] = acc;
        if (d == 0) p.part_ml[2 * part] = M, p.part_ml[2 * part + 1] = L;
    }
}

// o = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c over the chunks of a query head.
template <typename T, int D>
__global__ void __launch_bounds__(D) merge_kv8_kernel(const AttnKv8Params p) {
    pdl_wait();
    pdl_launch_dependents();
    const size_t row = blockIdx.x;
    const int d = threadIdx.x;
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int c = 0; c < p.chunks; ++c) M = fmaxf(M, p.part_ml[2 * (row * p.chunks + c)]);
    for (int c = 0; c < p.chunks; ++c) {
        const float m = p.part_ml[2 * (row * p.chunks + c)];
        const float w = m == -INFINITY ? 0.f : fast_exp2(m - M);
        L += w * p.part_ml[2 * (row * p.chunks + c) + 1];
        acc += w * p.part_o[(row * p.chunks + c) * D + d];
    }
    reinterpret_cast<T*>(p.o)[row * D + d] = from_f32<T>(L == 0.f ? 0.f : acc / L);
    if (p.lse && d == 0) p.lse[row] = L == 0.f ? -INFINITY : (M + log2f(L)) / kLog2e;
}

template <typename T, int D>
static int launch_attn_kv8(const AttnKv8Params& p, int batch, cudaStream_t st) {
    TIDAL_CUDA_OK(launch_pdl(attn_kv8_kernel<T, D>, dim3(p.chunks, batch * p.Hq), dim3(kKv8Warps * 32), 0, st, 1, p));
    TIDAL_CUDA_OK(launch_pdl(merge_kv8_kernel<T, D>, dim3(batch * p.Hq), dim3(D), 0, st, 1, p));
    count_launch(2);
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
    p.chunks = tidal_plan_chunks(a->batch, a->num_qo_heads, ntok, 64, 4 * sm_count_cached());
    p.sm_scale = a->sm_scale > 0.f ? a->sm_scale : 1.0f / sqrtf((float)a->head_dim);
    TIDAL_REQUIRE((int64_t)a->batch * a->num_qo_heads <= 65535, TIDAL_ERR_ARG, "batch * num_qo_heads beyond 65535");
    const size_t rows = (size_t)a->batch * a->num_qo_heads * p.chunks;
    TIDAL_REQUIRE(L->part_o_off + sizeof(float) * rows * a->head_dim <= L->part_ml_off && L->part_ml_off + sizeof(float) * rows * 2 <= L->hist_off,
                  TIDAL_ERR_WORKSPACE, "workspace was sized for a smaller batch/heads/head_dim than this call");
    cudaStream_t st = (cudaStream_t)stream;
    const bool wide = a->head_dim == 128;
    switch (a->dtype) {
        case TIDAL_DTYPE_F16: return wide ? launch_attn_kv8<__half, 128>(p, a->batch, st) : launch_attn_kv8<__half, 64>(p, a->batch, st);
        case TIDAL_DTYPE_BF16: return wide ? launch_attn_kv8<__nv_bfloat16, 128>(p, a->batch, st) : launch_attn_kv8<__nv_bfloat16, 64>(p, a->batch, st);
        default: return wide ? launch_attn_kv8<float, 128>(p, a->batch, st) : launch_attn_kv8<float, 64>(p, a->batch, st);
    }
}
