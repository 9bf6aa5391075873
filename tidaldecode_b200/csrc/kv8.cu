// Writing and reading an 8-bit KV pool: quantised append of new tokens, and read-back as 16/32-bit rows.
#include "kv8.cuh"

namespace tidal {

struct AppendKv8Params {
    const void* src[2];          // K rows, V rows
    int64_t stride[2];
    uint8_t* kv;
    uint8_t* scales;
    SlotMap map;
    const int32_t* pos0_dev;
    int32_t pos0, T, Hkv, block, blocks_per_seq;
    int64_t units;
    uint32_t* status;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
    using V = Vec16<T>;
#pragma unroll
    for (int i = 0; i < 8; i += V::N) V::to_float(*reinterpret_cast<const uint4*>(p + i), x + i);
}
__device__ __forceinline__ float finite_max8(float m, const float* x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = fabsf(x[i]);
        m = a < INFINITY ? fmaxf(m, a) : m;              // false for NaN too
    }
    return m;
}
__device__ __forceinline__ uint2 codes8(const float* x, float inv) {
    return make_uint2(pack_e4m3(x[0] * inv, x[1] * inv) | pack_e4m3(x[2] * inv, x[3] * inv) << 16,
                      pack_e4m3(x[4] * inv, x[5] * inv) | pack_e4m3(x[6] * inv, x[7] * inv) << 16);
}

// One unit of work is the part of one (block of slots, plane, head) that the call touches: its largest element decides
// the scale, so a first pass over the rows finds it and a second one writes the codes.  D/8 lanes cover a row.  A warp
// takes a unit; with blocks of one token, where a unit is a single row, every group of D/8 lanes takes its own (ONE).
template <typename T, int D, bool ONE>
__global__ void __launch_bounds__(256) append_kv8_kernel(const AppendKv8Params p) {
    constexpr int LPR = D / 8, RPW = 32 / LPR;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, group = lane / LPR, d0 = (lane % LPR) * 8;
    int64_t u = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (ONE) u = u * RPW + group;
    const bool live = u < p.units;
    if (!live) u = p.units - 1;                          // lanes without work follow along, for the shuffles, and store nothing
    const int h = (int)(u % p.Hkv);
    u /= p.Hkv;
    const int plane = (int)(u & 1);
    u >>= 1;
    const int j = (int)(u % p.blocks_per_seq), b = (int)(u / p.blocks_per_seq);
    const int pos0 = p.pos0_dev ? p.pos0_dev[b] : p.pos0;
    const int64_t end = (int64_t)pos0 + p.T;
    const int64_t s0 = pos0 < 0 ? -1 : (int64_t)(pos0 / p.block + j) * p.block;      // first slot of the block
    bool ok = live && s0 < end;
    int entry = 0;
    int64_t page = -1;
    if (ok) {
        // a start read from the device may lie behind the row of the page table (or behind the sequence's own pages)
        if (s0 <= INT32_MAX - p.block && s0 / p.map.page_size < p.map.pt_stride) page = p.map.page_of(b, (int)s0, &entry);
        if (page < 0) {
            if (p.status && d0 == 0) atomicOr(p.status, TIDAL_DEV_BAD_INDEX);
            ok = false;
        }
    }
    const int lo = ok && pos0 > s0 ? (int)(pos0 - s0) : 0;                            // rows [0, lo) hold codes already,
    const int hi = ok ? (int)min((int64_t)p.block, end - s0) : 0;                     // rows [lo, hi) are new
    const T* src = reinterpret_cast<const T*>(p.src[plane]) + ((int64_t)b * p.T + (s0 - pos0)) * p.stride[plane] + (size_t)h * D + d0;
    const int per_page = p.map.page_size / p.block;
    const size_t row0 = ((size_t)(ok ? page : 0) * 2 + plane) * p.map.page_size + entry;
    uint8_t* dst = p.kv + (row0 * p.Hkv + h) * D + d0;
    uint8_t* scale = p.scales + (((size_t)(ok ? page : 0) * 2 + plane) * per_page + entry / p.block) * p.Hkv + h;
    const size_t pitch = (size_t)p.Hkv * D;
    constexpr int STEP = ONE ? 1 : RPW;
    const int first = ONE ? 0 : group;

    float amax = 0.f;
    for (int r = lo + first; r < hi; r += STEP) {
        float x[8];
        load8(src + r * p.stride[plane], x);
        amax = finite_max8(amax, x);
    }
#pragma unroll
    for (int off = 1; off < (ONE ? LPR : 32); off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    if (!ok) return;
    int e = scale_byte(amax);
    if (lo > 0) {
        const int before = *scale;
        if (before >= e) {
            e = before;
        } else {
            // 2^(before - e): below 2^-126 every code becomes zero anyway
            const float shrink = scale_value((uint32_t)max(127 + before - e, 0));
            for (int r = first; r < lo; r += STEP) {
                const uint2 old = *reinterpret_cast<const uint2*>(dst + r * pitch);
                float x[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = unpack_e4m3(((i < 2 ? old.x : old.y) >> (16 * (i & 1))) & 0xffffu);
                    x[2 * i] = f.x;
                    x[2 * i + 1] = f.y;
                }
                *reinterpret_cast<uint2*>(dst + r * pitch) = codes8(x, shrink);
            }
        }
    }
    const float inv = scale_value((uint32_t)(254 - e));                               // 2^-(e-127); e <= 247 for any finite float
    for (int r = lo + first; r < hi; r += STEP) {
        float x[8];
        load8(src + r * p.stride[plane], x);
        *reinterpret_cast<uint2*>(dst + r * pitch) = codes8(x, inv);
    }
    if (!ONE) __syncwarp();                              // every lane has read the old scale
    if (d0 == 0 && (ONE || group == 0)) *scale = (uint8_t)e;
}

struct ReadKv8Params {
    const uint8_t* kv;
    const uint8_t* scales;
    SlotMap map;
    const int32_t* seq_lens;
    void* out;
    int32_t start, n, Hkv, block;
    int64_t vecs;                // 8-element vectors of the whole output
    uint32_t* status;
};

template <typename T, int D>
__global__ void __launch_bounds__(256) read_kv8_kernel(const ReadKv8Params p) {
    using V = Vec16<T>;
    pdl_wait();
    pdl_launch_dependents();
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= p.vecs) return;
    const int per_tok = 2 * p.Hkv * (D / 8);
    const int64_t tok = i / per_tok;
    int v = (int)(i - tok * per_tok);
    const int b = (int)(tok / p.n), slot = p.start + (int)(tok - (int64_t)b * p.n);
    if (p.seq_lens && slot >= p.seq_lens[b]) return;
    int entry;
    const int64_t page = p.map.page_of(b, slot, &entry);
    if (page < 0) {
        if (p.status && v == 0) atomicOr(p.status, TIDAL_DEV_BAD_INDEX);
        return;
    }
    const int d0 = v % (D / 8) * 8;
    v /= D / 8;
    const int h = v % p.Hkv, plane = v / p.Hkv;
    const size_t row = ((size_t)page * 2 + plane) * p.map.page_size + entry;
    const uint2 c = *reinterpret_cast<const uint2*>(p.kv + (row * p.Hkv + h) * D + d0);
    const float scale = scale_value(p.scales[(((size_t)page * 2 + plane) * (p.map.page_size / p.block) + entry / p.block) * p.Hkv + h]);
    float x[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = unpack_e4m3(((k < 2 ? c.x : c.y) >> (16 * (k & 1))) & 0xffffu);
        x[2 * k] = f.x * scale;
        x[2 * k + 1] = f.y * scale;
    }
    // fp16 ends at 65504: a value that was there may have been rounded up to 65536 or more
    if (sizeof(T) == 2 && V::round(65504.f) == 65504.f) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = x[k] > 65504.f ? 65504.f : (x[k] < -65504.f ? -65504.f : x[k]);
    }
    uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + i * 8);
#pragma unroll
    for (int k = 0; k < 8; k += V::N) out[k / V::N] = V::from_float(x + k);
}

static int check_pool(const char* what, int batch, int heads, int head_dim, int page_size, int block, int dtype, int64_t num_pages) {
    TIDAL_REQUIRE(batch >= 1 && heads >= 1, TIDAL_ERR_ARG, "%s: bad batch/num_kv_heads", what);
    TIDAL_REQUIRE(head_dim == 64 || head_dim == 128, TIDAL_ERR_ARG, "%s: unsupported head_dim %d (built: 64, 128)", what, head_dim);
    TIDAL_REQUIRE(dtype >= 0 && dtype <= 2, TIDAL_ERR_ARG, "%s: unknown dtype %d", what, dtype);
    TIDAL_REQUIRE(page_size >= 1 && num_pages >= 1, TIDAL_ERR_ARG, "%s: bad page_size/num_pages", what);
    TIDAL_REQUIRE(block >= 1 && page_size % block == 0, TIDAL_ERR_ARG, "%s: block %d does not divide page_size %d", what, block, page_size);
    return TIDAL_OK;
}

template <typename F>
static int by_type(int dtype, int head_dim, F&& f) {
    switch (dtype) {
        case TIDAL_DTYPE_F16: return head_dim == 64 ? f((__half*)nullptr, std::integral_constant<int, 64>()) : f((__half*)nullptr, std::integral_constant<int, 128>());
        case TIDAL_DTYPE_BF16:
            return head_dim == 64 ? f((__nv_bfloat16*)nullptr, std::integral_constant<int, 64>()) : f((__nv_bfloat16*)nullptr, std::integral_constant<int, 128>());
        default: return head_dim == 64 ? f((float*)nullptr, std::integral_constant<int, 64>()) : f((float*)nullptr, std::integral_constant<int, 128>());
    }
}

}  // namespace tidal

using namespace tidal;

extern "C" int tidal_append_kv8(const tidal_append_kv8_args* a, void* stream) {
    TIDAL_REQUIRE(a != nullptr, TIDAL_ERR_ARG, "args is NULL");
    TIDAL_REQUIRE(a->d_k && a->d_v && a->d_kv && a->d_scales, TIDAL_ERR_ARG, "append_kv8: k, v, kv and scales must be given");
    int rc = check_pool("append_kv8", a->batch, a->num_kv_heads, a->head_dim, a->page_size, a->block, a->dtype, a->num_pages);
    if (rc != TIDAL_OK) return rc;
    TIDAL_REQUIRE(a->tokens_per_seq >= 1, TIDAL_ERR_ARG, "append_kv8: bad tokens_per_seq %d", a->tokens_per_seq);
    TIDAL_REQUIRE(a->d_pos0 || (a->pos0 >= 0 && (int64_t)a->pos0 + a->tokens_per_seq <= INT32_MAX - a->block), TIDAL_ERR_ARG,
                  "append_kv8: bad pos0 %d", a->pos0);
    const int vec = a->dtype == TIDAL_DTYPE_F32 ? 4 : 8;
    TIDAL_REQUIRE((((uintptr_t)a->d_k | (uintptr_t)a->d_v | (uintptr_t)a->d_kv) & 15) == 0 && a->k_stride % vec == 0 && a->v_stride % vec == 0,
                  TIDAL_ERR_ARG, "append_kv8: rows of k, v and kv must be 16-byte aligned");
    TIDAL_REQUIRE(a->page_table_stride >= 1, TIDAL_ERR_ARG, "append_kv8: bad page_table_stride");
    if (!a->d_pos0) {
        const int64_t last = ((int64_t)a->pos0 + a->tokens_per_seq + a->page_size - 1) / a->page_size;      // pages of the longest sequence
        TIDAL_REQUIRE(last <= a->page_table_stride, TIDAL_ERR_ARG, "append_kv8: slots up to %lld need %lld pages, a sequence has %lld",
                      (long long)a->pos0 + a->tokens_per_seq, (long long)last, (long long)a->page_table_stride);
        TIDAL_REQUIRE(a->d_page_table || (int64_t)(a->batch - 1) * a->page_table_stride + last <= a->num_pages, TIDAL_ERR_ARG,
                      "append_kv8: identity page mapping runs past the pool's %lld pages", (long long)a->num_pages);
    }
    AppendKv8Params p;
    p.src[0] = a->d_k; p.src[1] = a->d_v;
    p.stride[0] = a->k_stride; p.stride[1] = a->v_stride;
    p.kv = (uint8_t*)a->d_kv; p.scales = a->d_scales;
    p.map = SlotMap{a->d_page_table, a->page_table_stride, a->num_pages, a->page_size};
    p.pos0_dev = a->d_pos0; p.pos0 = a->pos0; p.T = a->tokens_per_seq; p.Hkv = a->num_kv_heads; p.block = a->block;
    // with starts on the device the first block may be entered at any slot
    const int64_t lead = a->d_pos0 ? a->block - 1 : a->pos0 % a->block;
    p.blocks_per_seq = (int)((lead + a->tokens_per_seq + a->block - 1) / a->block);
    p.units = (int64_t)a->batch * p.blocks_per_seq * 2 * a->num_kv_heads;
    p.status = a->d_status;
    const int64_t per_cta = 8 * (a->block == 1 ? 32 / (a->head_dim / 8) : 1);
    const int64_t ctas = (p.units + per_cta - 1) / per_cta;
    TIDAL_REQUIRE(ctas <= INT32_MAX, TIDAL_ERR_ARG, "append_kv8: too many tokens for one call");
    rc = by_type(a->dtype, a->head_dim, [&](auto* t, auto d) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int D = decltype(d)::value;
        if (a->block == 1) TIDAL_CUDA_OK(launch_pdl(append_kv8_kernel<T, D, true>, dim3((unsigned)ctas), dim3(256), 0, (cudaStream_t)stream, 1, p));
        else TIDAL_CUDA_OK(launch_pdl(append_kv8_kernel<T, D, false>, dim3((unsigned)ctas), dim3(256), 0, (cudaStream_t)stream, 1, p));
        return TIDAL_OK;
    });
    if (rc == TIDAL_OK) count_launch();
    return rc;
}

extern "C" int tidal_read_kv8(const tidal_read_kv8_args* a, void* stream) {
    TIDAL_REQUIRE(a != nullptr, TIDAL_ERR_ARG, "args is NULL");
    TIDAL_REQUIRE(a->d_kv && a->d_scales && a->d_out, TIDAL_ERR_ARG, "read_kv8: kv, scales and out must be given");
    int rc = check_pool("read_kv8", a->batch, a->num_kv_heads, a->head_dim, a->page_size, a->block, a->dtype, a->num_pages);
    if (rc != TIDAL_OK) return rc;
    TIDAL_REQUIRE(a->start >= 0 && a->stop >= a->start, TIDAL_ERR_ARG, "read_kv8: bad range [%d, %d)", a->start, a->stop);
    TIDAL_REQUIRE((((uintptr_t)a->d_kv | (uintptr_t)a->d_out) & 15) == 0, TIDAL_ERR_ARG, "read_kv8: kv and out must be 16-byte aligned");
    const int64_t pages = ((int64_t)a->stop + a->page_size - 1) / a->page_size;
    TIDAL_REQUIRE(!a->d_page_table || pages <= a->page_table_stride, TIDAL_ERR_ARG, "read_kv8: slot %d lies behind the page table", a->stop);
    TIDAL_REQUIRE(a->d_page_table || (a->page_table_stride >= 0 && (int64_t)(a->batch - 1) * a->page_table_stride + pages <= a->num_pages), TIDAL_ERR_ARG,
                  "read_kv8: identity page mapping runs past the pool's %lld pages", (long long)a->num_pages);
    if (a->stop == a->start) return TIDAL_OK;
    ReadKv8Params p;
    p.kv = (const uint8_t*)a->d_kv; p.scales = a->d_scales;
    p.map = SlotMap{a->d_page_table, a->page_table_stride, a->num_pages, a->page_size};
    p.seq_lens = a->d_seq_lens; p.out = a->d_out; p.start = a->start; p.n = a->stop - a->start;
    p.Hkv = a->num_kv_heads; p.block = a->block; p.status = a->d_status;
    p.vecs = (int64_t)a->batch * p.n * 2 * a->num_kv_heads * (a->head_dim / 8);
    const int64_t ctas = (p.vecs + 255) / 256;
    TIDAL_REQUIRE(ctas <= INT32_MAX, TIDAL_ERR_ARG, "read_kv8: too many tokens for one call");
    rc = by_type(a->dtype, a->head_dim, [&](auto* t, auto d) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        TIDAL_CUDA_OK(launch_pdl(read_kv8_kernel<T, decltype(d)::value>, dim3((unsigned)ctas), dim3(256), 0, (cudaStream_t)stream, 1, p));
        return TIDAL_OK;
    });
    if (rc == TIDAL_OK) count_launch();
    return rc;
}
