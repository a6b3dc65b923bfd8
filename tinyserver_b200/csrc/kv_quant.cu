// Quantised paged KV cache: rows quantised as they are written to their
// pages, and read back as dense rows.  The arithmetic is in qf_quant.cuh.
//
// Store, per (token, head) row of K and of V: read D values, find the largest
// magnitude, write D codes and one fp32 scale.  Load: read codes and scale,
// write rnd(code * scale).  Both are bounded by HBM: 2 (D * es + D + 4) bytes
// per (token, head), es the element size.
//
// A thread owns 16 consecutive values of one K row and the same of the V row
// (64 to 128 bytes of loads in flight), D / 16 neighbouring lanes own a row,
// and the row maximum is log2(D / 16) shuffles.  A CTA takes one head of 256 /
// (D / 16) consecutive tokens, so that in a prefill, whose tokens fill
// consecutive slots of a page, its code rows and its 4-byte scales are whole
// sectors.  Rows of other widths, strides or alignments take one warp per row
// and element-wise accesses.
//
// 8 heads of 128, bf16 <-> e4m3, pages of 16 slots: 8192 tokens stored in 8.8 us (5.8
// TB/s), 16411 loaded in 19.0 us (5.4 TB/s); over int8, 256 tokens stored in 2.4 us and
// 484 loaded in 3.0 us, a launch's own time (0.3 us less by programmatic dependent launch).
#include "qf_quant.cuh"

namespace qf {
namespace {

struct QuantKv {
    const char* k_src;  // the dense rows: a store reads them through these
    const char* v_src;
    char* k_dst;  // and a load writes them through these
    char* v_dst;
    int64_t ks[3], vs[3];  // strides of those rows (head, token, dim), elements
    uint8_t* k_cache;
    uint8_t* v_cache;
    int64_t kc[4], vc[4];  // cache strides (block, head, slot, dim), codes
    float* k_scale;
    float* v_scale;
    int64_t kss[3], vss[3];  // scale strides (block, head, slot)
    const void* block_mapping;
    const void* slot_mapping;
    int index_type;
    int64_t T, Hkv, D, N, B;
    int32_t* status;
};

__device__ __forceinline__ bool place(const QuantKv& a, int64_t t, int64_t& blk, int64_t& slot,
                                      bool report) {
    blk = load_index(a.block_mapping, t, a.index_type);
    slot = load_index(a.slot_mapping, t, a.index_type);
    bool ok = true;
    if (blk < 0 || blk >= a.N) {
        if (report) flag(a.status, QF_FLAG_BAD_BLOCK);
        ok = false;
    }
    if (slot < 0 || slot >= a.B) {
        if (report) flag(a.status, QF_FLAG_BAD_SLOT);
        ok = false;
    }
    return ok;
}

// 16 values of a row as floats.
template <typename T>
__device__ __forceinline__ void load16(const char* p, float* f) {
    constexpr int PER = Dt<T>::kPerVec;
#pragma unroll
    for (int i = 0; i < 16 / PER; ++i) unpack<T>(ld_shared_ro16(p + 16 * i), f + PER * i);
}

// One row's codes and scale from 16 values per lane of its LPR lanes.
template <int FMT, int LPR>
__device__ __forceinline__ uint4 quantise16(const float* f, float& scale) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    float factor;
    row_scale<FMT>(m, scale, factor);
    uint4 c = make_uint4(0, 0, 0, 0);
    if (m < 0x7f800000u) {
        c.x = float_to_codes<FMT>(f[0] * factor, f[1] * factor, f[2] * factor, f[3] * factor);
        c.y = float_to_codes<FMT>(f[4] * factor, f[5] * factor, f[6] * factor, f[7] * factor);
        c.z = float_to_codes<FMT>(f[8] * factor, f[9] * factor, f[10] * factor, f[11] * factor);
        c.w = float_to_codes<FMT>(f[12] * factor, f[13] * factor, f[14] * factor, f[15] * factor);
    }
    return c;
}

template <typename T, int D, int FMT>
__global__ void __launch_bounds__(256) quant_store_kernel(const QuantKv a) {
    pdl_wait();
    pdl_trigger();
    constexpr int LPR = D / 16;     // lanes per row
    constexpr int TT = 256 / LPR;   // tokens per CTA
    constexpr int64_t ES = sizeof(T);
    const int c = threadIdx.x % LPR, r = threadIdx.x / LPR;
    const int64_t h = blockIdx.y;
    const int64_t t = (int64_t)blockIdx.x * TT + r;
    const bool live = t < a.T;
    const int64_t tt = live ? t : a.T - 1;  // every lane takes part in the shuffles
    float k[16], v[16];
    load16<T>(a.k_src + (h * a.ks[0] + tt * a.ks[1] + c * 16) * ES, k);
    load16<T>(a.v_src + (h * a.vs[0] + tt * a.vs[1] + c * 16) * ES, v);
    int64_t blk, slot;
    const bool ok = place(a, tt, blk, slot, live && c == 0 && h == 0);
    float sk, sv;
    const uint4 ck = quantise16<FMT, LPR>(k, sk);
    const uint4 cv = quantise16<FMT, LPR>(v, sv);
    if (!live || !ok) return;
    st16(a.k_cache + blk * a.kc[0] + h * a.kc[1] + slot * a.kc[2] + c * 16, ck);
    st16(a.v_cache + blk * a.vc[0] + h * a.vc[1] + slot * a.vc[2] + c * 16, cv);
    if (c == 0) {
        a.k_scale[blk * a.kss[0] + h * a.kss[1] + slot * a.kss[2]] = sk;
        a.v_scale[blk * a.vss[0] + h * a.vss[1] + slot * a.vss[2]] = sv;
    }
}

template <typename T, int FMT>
__device__ __forceinline__ void dequantise16(char* dst, const uint4& c, float scale) {
    float f[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) codes_to_float<FMT>(word(c, i), f + 4 * i);
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] *= scale;
    constexpr int PER = Dt<T>::kPerVec;
#pragma unroll
    for (int i = 0; i < 16 / PER; ++i) st16(dst + 16 * i, pack<T>(f + PER * i));
}

template <typename T, int D, int FMT>
__global__ void __launch_bounds__(256) quant_load_kernel(const QuantKv a) {
    pdl_wait();
    pdl_trigger();
    constexpr int LPR = D / 16, TT = 256 / LPR;
    constexpr int64_t ES = sizeof(T);
    const int c = threadIdx.x % LPR, r = threadIdx.x / LPR;
    const int64_t h = blockIdx.y;
    const int64_t t = (int64_t)blockIdx.x * TT + r;
    if (t >= a.T) return;
    int64_t blk, slot;
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    float sk = 0.f, sv = 0.f;  // a place outside the cache reads as zeros
    if (place(a, t, blk, slot, c == 0 && h == 0)) {
        k = ld_shared_ro16(a.k_cache + blk * a.kc[0] + h * a.kc[1] + slot * a.kc[2] + c * 16);
        v = ld_shared_ro16(a.v_cache + blk * a.vc[0] + h * a.vc[1] + slot * a.vc[2] + c * 16);
        sk = __ldg(a.k_scale + blk * a.kss[0] + h * a.kss[1] + slot * a.kss[2]);
        sv = __ldg(a.v_scale + blk * a.vss[0] + h * a.vss[1] + slot * a.vss[2]);
    }
    dequantise16<T, FMT>(a.k_dst + (h * a.ks[0] + t * a.ks[1] + c * 16) * ES, k, sk);
    dequantise16<T, FMT>(a.v_dst + (h * a.vs[0] + t * a.vs[1] + c * 16) * ES, v, sv);
}

// One warp per (token, head) row of K or V: any width, stride and alignment.
template <typename T, int FMT, bool STORE>
__global__ void __launch_bounds__(256) quant_row_kernel(const QuantKv a) {
    const int lane = threadIdx.x & 31;
    const int64_t rows = a.T * a.Hkv;
    const int64_t step = (int64_t)gridDim.x * 8;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < rows; i += step) {
        const int64_t t = i / a.Hkv, h = i - t * a.Hkv;
        int64_t blk, slot;
        const bool ok = place(a, t, blk, slot, lane == 0 && h == 0);
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const int64_t* ss = side ? a.vs : a.ks;
            const int64_t* cs = side ? a.vc : a.kc;
            const int64_t* sc = side ? a.vss : a.kss;
            uint8_t* cache = (side ? a.v_cache : a.k_cache) + (ok ? blk * cs[0] + h * cs[1] + slot * cs[2] : 0);
            float* scales = (side ? a.v_scale : a.k_scale) + (ok ? blk * sc[0] + h * sc[1] + slot * sc[2] : 0);
            if constexpr (STORE) {
                if (!ok) continue;
                const T* src = reinterpret_cast<const T*>(side ? a.v_src : a.k_src) + h * ss[0] + t * ss[1];
                uint32_t m = 0;
                for (int64_t d = lane; d < a.D; d += 32)
                    m = max(m, __float_as_uint(Dt<T>::to_f(src[d * ss[2]])) & 0x7fffffffu);
                m = __reduce_max_sync(0xffffffffu, m);
                float scale, factor;
                row_scale<FMT>(m, scale, factor);
                for (int64_t d = lane; d < a.D; d += 32) {
                    const float x = m < 0x7f800000u ? Dt<T>::to_f(src[d * ss[2]]) * factor : 0.f;
                    cache[d * cs[3]] = (uint8_t)float_to_codes<FMT>(x, 0.f, 0.f, 0.f);
                }
                if (lane == 0) *scales = scale;
            } else {
                T* dst = reinterpret_cast<T*>(side ? a.v_dst : a.k_dst) + h * ss[0] + t * ss[1];
                const float scale = ok ? *scales : 0.f;
                for (int64_t d = lane; d < a.D; d += 32)
                    dst[d * ss[2]] = Dt<T>::from_f(ok ? code_to_float<FMT>(cache[d * cs[3]]) * scale : 0.f);
            }
        }
    }
}

template <typename T, int FMT, bool STORE>
int launch(const QuantKv& a, bool fast, cudaStream_t stream) {
    if (fast) {
        const int64_t tt = 256 / (a.D / 16);
        const dim3 grid((unsigned)ceil_div(a.T, tt), (unsigned)a.Hkv);
#define QF_QUANT_CASE(DD)                                                            \
    case DD:                                                                         \
        if constexpr (STORE) return launch_pdl(quant_store_kernel<T, DD, FMT>, grid, 256, 0, stream, a); \
        else return launch_pdl(quant_load_kernel<T, DD, FMT>, grid, 256, 0, stream, a);
        switch (a.D) {
            QF_QUANT_CASE(64)
            QF_QUANT_CASE(128)
            QF_QUANT_CASE(256)
        }
#undef QF_QUANT_CASE
    }
    const int64_t ctas = std::min<int64_t>(ceil_div(a.T * a.Hkv, 8), (int64_t)sm_count() * 8);
    quant_row_kernel<T, FMT, STORE><<<(unsigned)ctas, 256, 0, stream>>>(a);
    return check_launch();
}

template <bool STORE>
int run(const qf_kv_quantized_args* p, cudaStream_t stream) {
    if (!p) return QF_ERR_INVALID;
    const qf_kv_quantized_args& g = *p;
    if (g.num_tokens < 0 || g.num_kv_heads < 0 || g.head_dim < 0 || g.num_blocks < 0 ||
        g.block_size < 0)
        return QF_ERR_INVALID;
    if (g.index_type != QF_I32 && g.index_type != QF_I64) return QF_ERR_INVALID;
    if (g.dtype != QF_F32 && g.dtype != QF_F16 && g.dtype != QF_BF16) return QF_ERR_INVALID;
    if (g.format != QF_CACHE_E4M3 && g.format != QF_CACHE_INT8) return QF_ERR_INVALID;
    const int64_t D = g.head_dim;
    if (g.num_tokens == 0 || g.num_kv_heads == 0 || D == 0) return QF_OK;
    if (!g.k_rows || !g.v_rows || !g.k_cache || !g.v_cache || !g.k_scale || !g.v_scale ||
        !g.block_mapping || !g.slot_mapping)
        return QF_ERR_INVALID;
    if (g.num_tokens > ((int64_t)1 << 31) || g.num_kv_heads > 65535) return QF_ERR_UNSUPPORTED;
    QuantKv a{};
    a.k_src = a.k_dst = static_cast<char*>(g.k_rows);
    a.v_src = a.v_dst = static_cast<char*>(g.v_rows);
    a.k_cache = static_cast<uint8_t*>(g.k_cache);
    a.v_cache = static_cast<uint8_t*>(g.v_cache);
    a.k_scale = g.k_scale;
    a.v_scale = g.v_scale;
    const int64_t es = g.dtype == QF_F32 ? 4 : 2;
    // 16-byte accesses: whole rows contiguous, every row start a multiple of 16 bytes
    bool fast = (D == 64 || D == 128 || D == 256) && aligned16(g.k_rows) && aligned16(g.v_rows) &&
                aligned16(g.k_cache) && aligned16(g.v_cache) && g.k_row_strides[2] == 1 &&
                g.v_row_strides[2] == 1 && g.k_cache_strides[3] == 1 && g.v_cache_strides[3] == 1;
    for (int i = 0; i < 3; ++i) {
        a.ks[i] = g.k_row_strides[i];
        a.vs[i] = g.v_row_strides[i];
        a.kss[i] = g.k_scale_strides[i];
        a.vss[i] = g.v_scale_strides[i];
        if (i < 2) fast = fast && (a.ks[i] * es) % 16 == 0 && (a.vs[i] * es) % 16 == 0;
    }
    for (int i = 0; i < 4; ++i) {
        a.kc[i] = g.k_cache_strides[i];
        a.vc[i] = g.v_cache_strides[i];
        if (i < 3) fast = fast && a.kc[i] % 16 == 0 && a.vc[i] % 16 == 0;
    }
    a.block_mapping = g.block_mapping;
    a.slot_mapping = g.slot_mapping;
    a.index_type = g.index_type;
    a.T = g.num_tokens;
    a.Hkv = g.num_kv_heads;
    a.D = D;
    a.N = g.num_blocks;
    a.B = g.block_size;
    a.status = g.status;
    const bool e4m3 = g.format == QF_CACHE_E4M3;
    switch (g.dtype) {
    case QF_F32:
        return e4m3 ? launch<float, QF_CACHE_E4M3, STORE>(a, fast, stream)
                    : launch<float, QF_CACHE_INT8, STORE>(a, fast, stream);
    case QF_F16:
        return e4m3 ? launch<__half, QF_CACHE_E4M3, STORE>(a, fast, stream)
                    : launch<__half, QF_CACHE_INT8, STORE>(a, fast, stream);
    default:
        return e4m3 ? launch<__nv_bfloat16, QF_CACHE_E4M3, STORE>(a, fast, stream)
                    : launch<__nv_bfloat16, QF_CACHE_INT8, STORE>(a, fast, stream);
    }
}

}  // namespace
}  // namespace qf

extern "C" int qf_kv_store_quantized(const qf_kv_quantized_args* args, cudaStream_t stream) {
    return qf::run<true>(args, stream);
}

extern "C" int qf_kv_load_quantized(const qf_kv_quantized_args* args, cudaStream_t stream) {
    return qf::run<false>(args, stream);
}

extern "C" size_t qf_kv_quantized_args_size(void) { return sizeof(qf_kv_quantized_args); }
