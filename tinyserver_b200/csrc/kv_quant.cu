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
        if constexpr (STORE) quant_store_kernel<T, DD, FMT><<<grid, 256, 0, stream>>>(a); \
        else quant_load_kernel<T, DD, FMT><<<grid, 256, 0, stream>>>(a);             \
        return check_launch();
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
int run(const void* k_rows, const int64_t* ks, const void* v_rows, const int64_t* vs, const void* k_cache,
        const int64_t* kc, const void* v_cache, const int64_t* vc, const void* k_scale,
        const int64_t* kss, const void* v_scale, const int64_t* vss, const void* block_mapping,
        const void* slot_mapping, int index_type, int64_t T, int64_t Hkv, int64_t D, int64_t N,
        int64_t B, int dtype, int format, int32_t* status, cudaStream_t stream) {
    if (T < 0 || Hkv < 0 || D < 0 || N < 0 || B < 0) return QF_ERR_INVALID;
    if (index_type != QF_I32 && index_type != QF_I64) return QF_ERR_INVALID;
    if (dtype != QF_F32 && dtype != QF_F16 && dtype != QF_BF16) return QF_ERR_INVALID;
    if (format != QF_CACHE_E4M3 && format != QF_CACHE_INT8) return QF_ERR_INVALID;
    if (T == 0 || Hkv == 0 || D == 0) return QF_OK;
    if (!k_rows || !v_rows || !k_cache || !v_cache || !k_scale || !v_scale || !block_mapping ||
        !slot_mapping || !ks || !vs || !kc || !vc || !kss || !vss)
        return QF_ERR_INVALID;
    if (T > ((int64_t)1 << 31) || Hkv > 65535) return QF_ERR_UNSUPPORTED;
    QuantKv a{};
    a.k_src = static_cast<const char*>(k_rows);
    a.v_src = static_cast<const char*>(v_rows);
    a.k_dst = static_cast<char*>(const_cast<void*>(k_rows));
    a.v_dst = static_cast<char*>(const_cast<void*>(v_rows));
    a.k_cache = static_cast<uint8_t*>(const_cast<void*>(k_cache));
    a.v_cache = static_cast<uint8_t*>(const_cast<void*>(v_cache));
    a.k_scale = static_cast<float*>(const_cast<void*>(k_scale));
    a.v_scale = static_cast<float*>(const_cast<void*>(v_scale));
    const int64_t es = dtype == QF_F32 ? 4 : 2;
    // 16-byte accesses: whole rows contiguous, every row start a multiple of 16 bytes
    bool fast = (D == 64 || D == 128 || D == 256) && aligned16(k_rows) && aligned16(v_rows) &&
                aligned16(k_cache) && aligned16(v_cache) && ks[2] == 1 && vs[2] == 1 &&
                kc[3] == 1 && vc[3] == 1;
    for (int i = 0; i < 3; ++i) {
        a.ks[i] = ks[i];
        a.vs[i] = vs[i];
        a.kss[i] = kss[i];
        a.vss[i] = vss[i];
        if (i < 2) fast = fast && (ks[i] * es) % 16 == 0 && (vs[i] * es) % 16 == 0;
    }
    for (int i = 0; i < 4; ++i) {
        a.kc[i] = kc[i];
        a.vc[i] = vc[i];
        if (i < 3) fast = fast && kc[i] % 16 == 0 && vc[i] % 16 == 0;
    }
    a.block_mapping = block_mapping;
    a.slot_mapping = slot_mapping;
    a.index_type = index_type;
    a.T = T;
    a.Hkv = Hkv;
    a.D = D;
    a.N = N;
    a.B = B;
    a.status = status;
    const bool e4m3 = format == QF_CACHE_E4M3;
    switch (dtype) {
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

extern "C" int qf_kv_store_quantized(
    const void* k_src, const int64_t k_src_strides[3], const void* v_src,
    const int64_t v_src_strides[3], void* k_cache, const int64_t k_cache_strides[4], void* v_cache,
    const int64_t v_cache_strides[4], float* k_scale, const int64_t k_scale_strides[3],
    float* v_scale, const int64_t v_scale_strides[3], const void* block_mapping,
    const void* slot_mapping, int index_type, int64_t num_tokens, int64_t num_kv_heads,
    int64_t head_dim, int64_t num_blocks, int64_t block_size, int dtype, int format,
    int32_t* status, cudaStream_t stream) {
    return qf::run<true>(k_src, k_src_strides, v_src, v_src_strides, k_cache, k_cache_strides,
                         v_cache, v_cache_strides, k_scale, k_scale_strides, v_scale,
                         v_scale_strides, block_mapping, slot_mapping, index_type, num_tokens,
                         num_kv_heads, head_dim, num_blocks, block_size, dtype, format, status,
                         stream);
}

extern "C" int qf_kv_load_quantized(
    const void* k_cache, const int64_t k_cache_strides[4], const void* v_cache,
    const int64_t v_cache_strides[4], const float* k_scale, const int64_t k_scale_strides[3],
    const float* v_scale, const int64_t v_scale_strides[3], const void* block_mapping,
    const void* slot_mapping, int index_type, void* k_out, const int64_t k_out_strides[3],
    void* v_out, const int64_t v_out_strides[3], int64_t num_tokens, int64_t num_kv_heads,
    int64_t head_dim, int64_t num_blocks, int64_t block_size, int dtype, int format,
    int32_t* status, cudaStream_t stream) {
    return qf::run<false>(k_out, k_out_strides, v_out, v_out_strides, k_cache, k_cache_strides,
                          v_cache, v_cache_strides, k_scale, k_scale_strides, v_scale,
                          v_scale_strides, block_mapping, slot_mapping, index_type, num_tokens,
                          num_kv_heads, head_dim, num_blocks, block_size, dtype, format, status,
                          stream);
}
