// Writing and reading an 8-bit KV pool: quantised append of new tokens, and read-back as 16/32-bit rows.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "kv8.cuh"

namespace tidal {

struct AppendKv8Params {
    const void* src[2];          // K rows, V rows
    int64_t stride[2];
    uint8_t* kv;
    uint8_t* scales;
    SlotMap map;
    const int32_t* pos0_dev;
    int32_t pos0, T, Hkv, block, blocks_per_page, blocks_per_seq;
    uint32_t units;
    uint32_t* status;
};

// Eight elements of a row as they are stored, and as floats.
template <typename T>
struct Raw8 {
    uint4 v[8 / Vec16<T>::N];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < 8 / Vec16<T>::N; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void floats(float* x) const {
#pragma unroll
        for (int i = 0; i < 8 / Vec16<T>::N; ++i) Vec16<T>::to_float(v[i], x + i * Vec16<T>::N);
    }
};
// Running maximum of the magnitudes, in pairs where the type has pairs: NaN is left out by the instruction, infinities are
// looked for at the end.
template <typename T>
struct AbsMax;
template <>
struct AbsMax<__half> {
    __half2 m = __half2half2(__ushort_as_half(0));
    __device__ __forceinline__ void add(const Raw8<__half>& r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __hmax2(m, __habs2(reinterpret_cast<const __half2*>(&r.v[0])[i]));
    }
    __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};
template <>
struct AbsMax<__nv_bfloat16> {
    __nv_bfloat162 m = __bfloat162bfloat162(__ushort_as_bfloat16(0));
    __device__ __forceinline__ void add(const Raw8<__nv_bfloat16>& r) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __hmax2(m, __habs2(reinterpret_cast<const __nv_bfloat162*>(&r.v[0])[i]));
    }
    __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};
template <>
struct AbsMax<float> {
    float m = 0.f;
    __device__ __forceinline__ void add(const Raw8<float>& r) {
        float x[8];
        r.floats(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i]));
    }
    __device__ __forceinline__ float get() const { return m; }
};
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
// Codes of eight stored elements times inv, a power of two.  fp16 rows stay in pairs while inv is an fp16 number (2^-24 ..
// 2^15; the scale of a block that holds tokens of another type may ask for less): the product is exact, or below 2^-14 and
// then a zero code either way.
template <typename T>
__device__ __forceinline__ uint2 codes8(const Raw8<T>& r, float inv) {
    if (std::is_same<T, __half>::value && inv >= 0x1p-24f && inv <= 0x1p15f) {
        const __half2 k = __float2half2_rn(inv);
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 y = __hmul2(reinterpret_cast<const __half2*>(&r.v[0])[i], k);
            c[i] = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(y), __NV_SATFINITE, __NV_E4M3);
        }
        return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
    }
    float x[8];
    r.floats(x);
    return codes8(x, inv);
}
__device__ __forceinline__ void values8(uint2 c, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_e4m3(((i < 2 ? c.x : c.y) >> (16 * (i & 1))) & 0xffffu);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// One unit of work is the part of one (block of slots, plane, head) that the call touches: its largest element decides
// the scale of all its codes.  D/8 lanes cover a row.  A warp takes a unit; with blocks of one token, where a unit is a
// single row, every group of D/8 lanes takes its own (ONE).  Up to eight (32-bit rows: four) row steps stay in registers between the pass that
// finds the maximum and the one that writes codes, with all their loads in flight at once; longer blocks read the rows
// behind those a second time (from L2).  Bound by HBM: 16-bit rows in, 8-bit codes out.  32 K tokens x 32 heads x 128, fp16,
// blocks of 16: 158 us for 805 MB, 5.1 TB/s (a sixth more while the rows waited for the page lookup).
template <typename T, int D, bool ONE>
__global__ void __launch_bounds__(256) append_kv8_kernel(const AppendKv8Params p) {
    constexpr int LPR = D / 8, RPW = 32 / LPR;
    constexpr int STEP = ONE ? 1 : RPW, HELD = ONE ? 1 : sizeof(T) == 4 ? 4 : 8;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, group = lane / LPR, d0 = (lane % LPR) * 8;
    uint32_t u = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (ONE) u = u * RPW + group;
    const bool live = u < p.units;
    if (!live) u = p.units - 1;                          // lanes without work follow along, for the shuffles, and store nothing
    const uint32_t rest = u / (uint32_t)p.Hkv;
    const int h = (int)(u - rest * (uint32_t)p.Hkv), plane = (int)(rest & 1);
    const int b = (int)((rest >> 1) / (uint32_t)p.blocks_per_seq), j = (int)((rest >> 1) - (uint32_t)b * (uint32_t)p.blocks_per_seq);
    const int pos0 = p.pos0_dev ? p.pos0_dev[b] : p.pos0;
    const int64_t end = (int64_t)pos0 + p.T;
    const int64_t s0 = pos0 < 0 ? -1 : ((int64_t)(pos0 / p.block) + j) * p.block;    // first slot of the block (a start may be any number)
    const bool in = live && pos0 >= 0 && s0 < end && s0 <= INT32_MAX - p.block;
    const int lo = in && pos0 > s0 ? (int)(pos0 - s0) : 0;                            // rows [0, lo) hold codes already,
    const int hi = in ? (int)min((int64_t)p.block, end - s0) : 0;                     // rows [lo, hi) are new
    const T* src = reinterpret_cast<const T*>(p.src[plane]) + ((int64_t)b * p.T + (s0 - pos0)) * p.stride[plane] + (size_t)h * D + d0;
    const int first = lo + (ONE ? 0 : group);
    Raw8<T> held[HELD];                                  // on their way before the page is known
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (first + i * STEP < hi) held[i].load(src + (first + i * STEP) * p.stride[plane]);
    bool ok = in;
    int entry = 0;
    int64_t page = -1;
    // a start read from the device may lie behind the row of the page table (or behind the sequence's own pages)
    if (in && (int)s0 / p.map.page_size < p.map.pt_stride) page = p.map.page_of(b, (int)s0, &entry);
    if (page < 0) {
        if (live && (pos0 < 0 || s0 < end) && p.status && d0 == 0) atomicOr(p.status, TIDAL_DEV_BAD_INDEX);
        ok = false;
    }
    const size_t row0 = ((size_t)(ok ? page : 0) * 2 + plane) * p.map.page_size + entry;
    uint8_t* dst = p.kv + (row0 * p.Hkv + h) * D + d0;
    uint8_t* scale = p.scales + (((size_t)(ok ? page : 0) * 2 + plane) * p.blocks_per_page + (p.blocks_per_page > 1 ? entry / p.block : 0)) * p.Hkv + h;
    const size_t pitch = (size_t)p.Hkv * D;
    const int before = ok && lo > 0 ? *scale : 0;
    float x[8];
    AbsMax<T> top;
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (first + i * STEP < hi) top.add(held[i]);
    if (!ONE)
        for (int r = first + HELD * STEP; r < hi; r += STEP) {
            Raw8<T> raw;
            raw.load(src + r * p.stride[plane]);
            top.add(raw);
        }
    float amax = top.get();
    if (__any_sync(0xffffffffu, amax == INFINITY)) {     // an infinity somewhere: the finite elements decide
        amax = 0.f;
        for (int r = first; r < hi; r += STEP) {
            Raw8<T> raw;
            raw.load(src + r * p.stride[plane]);
            raw.floats(x);
            amax = finite_max8(amax, x);
        }
    }
#pragma unroll
    for (int off = 1; off < (ONE ? LPR : 32); off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    if (!ok) return;
    int e = scale_byte(amax);
    if (lo > 0) {
        if (before >= e) {
            e = before;
        } else {
            // 2^(before - e): below 2^-126 every code becomes zero anyway
            const float shrink = scale_value((uint32_t)max(127 + before - e, 0));
            for (int r = group; r < lo; r += STEP) {
                values8(*reinterpret_cast<const uint2*>(dst + r * pitch), x);
                *reinterpret_cast<uint2*>(dst + r * pitch) = codes8(x, shrink);
            }
        }
    }
    const float inv = scale_value((uint32_t)(254 - e));                               // 2^-(e-127); e <= 247 for any finite float
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (first + i * STEP < hi) {
            *reinterpret_cast<uint2*>(dst + (first + i * STEP) * pitch) = codes8(held[i], inv);
        }
    if (!ONE) {
        for (int r = first + HELD * STEP; r < hi; r += STEP) {
            Raw8<T> raw;
            raw.load(src + r * p.stride[plane]);
            *reinterpret_cast<uint2*>(dst + r * pitch) = codes8(raw, inv);
        }
        __syncwarp();                                    // every lane has read the old scale
    }
    if (d0 == 0 && (ONE || group == 0)) *scale = (uint8_t)e;
}

struct ReadKv8Params {
    const uint8_t* kv;
    const uint8_t* scales;
    SlotMap map;
    const int32_t* seq_lens;
    void* out;
    int32_t start, n, Hkv, block, blocks_per_page;
    int32_t per_tok;             // 16-element vectors of a token (both planes, all heads)
    int32_t toks;                // tokens a CTA takes at a time: 256 / per_tok, at least one
    int32_t page_shift;          // -1: page_size is no power of two
    uint32_t* status;
};

// A thread keeps its plane, head and 16 elements and walks over tokens, kReadSteps of them with their loads in flight together.
// Bound by HBM: 32 K tokens x 32 heads x 128 to fp16, 131 us for 805 MB, 6.1 TB/s.  With all indices formed anew per vector it
// was bound by instructions (310 for 16 codes, 158 us).
constexpr int kReadSteps = 2;
template <typename T, int D>
__global__ void __launch_bounds__(256) read_kv8_kernel(const ReadKv8Params p) {
    using V = Vec16<T>;
    constexpr int VPR = D / 16;
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.y;
    const int sub = (int)threadIdx.x / p.per_tok;
    const int v = blockIdx.z * 256 + (p.toks > 1 ? (int)threadIdx.x - sub * p.per_tok : (int)threadIdx.x);
    if (v >= p.per_tok || (p.toks > 1 && sub >= p.toks)) return;
    const int hp = v / VPR, plane = hp >= p.Hkv ? 1 : 0, h = hp - plane * p.Hkv;
    const int last = p.seq_lens ? (int)min((int64_t)p.n, max((int64_t)p.seq_lens[b] - p.start, (int64_t)0)) : p.n;
    const int tok0 = (int)blockIdx.x * kReadSteps * p.toks + (p.toks > 1 ? sub : 0);
    const int32_t* table = p.map.page_table ? p.map.page_table + (size_t)b * p.map.pt_stride : nullptr;
    const int64_t page0 = (int64_t)b * p.map.pt_stride;
    const uint8_t* codes = p.kv + (size_t)h * D + v % VPR * 16;
    const uint8_t* scales = p.scales + h;
    const int ps = p.map.page_size;
    uint4 c[kReadSteps];
    uint32_t sc[kReadSteps];
    int64_t row[kReadSteps];
#pragma unroll
    for (int s = 0; s < kReadSteps; ++s) {
        const int tok = tok0 + s * p.toks;
        row[s] = -1;
        if (tok < last) {
            const int slot = p.start + tok, pg = p.page_shift >= 0 ? slot >> p.page_shift : slot / ps, entry = slot - pg * ps;
            const int64_t page = table ? (int64_t)table[pg] : page0 + pg;
            if (page >= 0 && page < p.map.num_pages) {
                row[s] = (page * 2 + plane) * ps + entry;
                const int blk = p.blocks_per_page > 1 ? entry / p.block : 0;
                sc[s] = scales[((page * 2 + plane) * p.blocks_per_page + blk) * p.Hkv];
                c[s] = *reinterpret_cast<const uint4*>(codes + (size_t)row[s] * (uint32_t)(p.Hkv * D));
            } else if (v == 0 && p.status) {
                atomicOr(p.status, TIDAL_DEV_BAD_INDEX);
            }
        }
    }
    T* out = reinterpret_cast<T*>(p.out) + ((size_t)b * p.n + tok0) * (p.per_tok * 16) + v * 16;
    const size_t step = (size_t)p.toks * p.per_tok * 16;
#pragma unroll
    for (int s = 0; s < kReadSteps; ++s) {
        if (row[s] < 0) continue;
        uint4* to = reinterpret_cast<uint4*>(out + s * step);
        if (std::is_same<T, __half>::value && sc[s] >= 103u && sc[s] <= 142u) {
            // the scale is an fp16 number (2^-24 .. 2^15): pairs stay pairs, one rounding as below.  fp16 ends at 65504; a value
            // that was there may have been rounded up to 65536 or more
            const __half2 k = __float2half2_rn(scale_value(sc[s])), top = __float2half2_rn(65504.f), low = __float2half2_rn(-65504.f);
            const uint32_t w[4] = {c[s].x, c[s].y, c[s].z, c[s].w};
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (16 * (i & 1)) & 0xffffu), __NV_E4M3);
                const __half2 y = __hmax2_nan(__hmin2_nan(__hmul2(*reinterpret_cast<const __half2*>(&r), k), top), low);
                o[i] = *reinterpret_cast<const uint32_t*>(&y);
            }
            to[0] = make_uint4(o[0], o[1], o[2], o[3]);
            to[1] = make_uint4(o[4], o[5], o[6], o[7]);
            continue;
        }
        float x[16];
        const float k = scale_value(sc[s]);
        values8(make_uint2(c[s].x, c[s].y), x);
        values8(make_uint2(c[s].z, c[s].w), x + 8);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= k;
        // 2^120, the scale of the largest floats, is the one at which 32-bit and bf16 rows can pass their type's end
        if (std::is_same<T, __half>::value || sc[s] >= 247u) {
            constexpr float most = std::is_same<T, __half>::value ? 65504.f : sizeof(T) == 4 ? FLT_MAX : 0x1.fep127f;
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = x[i] > most ? most : (x[i] < -most ? -most : x[i]);
        }
#pragma unroll
        for (int i = 0; i < 16; i += V::N) to[i / V::N] = V::from_float(x + i);
    }
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
    p.blocks_per_page = a->page_size / a->block;
    const int64_t units = (int64_t)a->batch * p.blocks_per_seq * 2 * a->num_kv_heads;
    TIDAL_REQUIRE(units <= INT32_MAX, TIDAL_ERR_ARG, "append_kv8: too many tokens for one call (%lld blocks and heads)", (long long)units);
    p.units = (uint32_t)units;
    p.status = a->d_status;
    const int64_t per_cta = 8 * (a->block == 1 ? 32 / (a->head_dim / 8) : 1);
    const int64_t ctas = (units + per_cta - 1) / per_cta;
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
    p.blocks_per_page = a->page_size / a->block;
    TIDAL_REQUIRE(a->num_kv_heads <= 1 << 16 && a->batch <= 65535, TIDAL_ERR_ARG, "read_kv8: too many heads or sequences for one call");
    p.per_tok = 2 * a->num_kv_heads * (a->head_dim / 16);
    p.toks = std::max(1, 256 / p.per_tok);
    p.page_shift = (a->page_size & (a->page_size - 1)) == 0 ? 31 - __builtin_clz((unsigned)a->page_size) : -1;
    const dim3 grid((unsigned)((p.n + (int64_t)kReadSteps * p.toks - 1) / (kReadSteps * p.toks)), a->batch, (p.per_tok + 255) / 256);
    rc = by_type(a->dtype, a->head_dim, [&](auto* t, auto d) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        TIDAL_CUDA_OK(launch_pdl(read_kv8_kernel<T, decltype(d)::value>, grid, dim3(256), 0, (cudaStream_t)stream, 1, p));
        return TIDAL_OK;
    });
    if (rc == TIDAL_OK) count_launch();
    return rc;
}
