// Shared by the kernels of attention over the paged cache for several new
// tokens per sequence (paged_tree*.cu): arguments, lengths, key addresses.
#pragma once

#include "qf_common.cuh"

namespace qf {

// j / d for 0 <= j < 2^31 by one 64-bit multiply and a shift: with
// m = ceil(2^(32 + s) / d), s = floor(log2 d), the quotient is exact there
// (m has at most 33 bits; the error j (m d - 2^(32+s)) / (d 2^(32+s)) < 1 / d).
struct FastDiv {
    uint64_t m;
    int s, d;
    FastDiv() = default;
    explicit FastDiv(int div) : d(div) {
        s = 0;
        while (s < 30 && (2ll << s) <= div) ++s;
        m = ((1ull << (32 + s)) + (uint64_t)div - 1) / (uint64_t)div;
    }
    __device__ __forceinline__ int div(int j) const {
        return (int)(((uint64_t)(uint32_t)j * m) >> (32 + s));
    }
};

struct TreeDev {
    const char* q;
    int64_t qt, qh;  // query strides (token, head), elements
    const char* kc;
    const char* vc;
    int64_t c0, c1, c2;  // cache strides (block, head, slot), elements
    const float* ks;
    const float* vs;
    int64_t s0, s1, s2;  // scale strides (block, head, slot)
    int64_t N;
    FastDiv B;
    const int32_t* bt;
    int64_t bts;
    int cap;  // keys a block-table row describes
    const int32_t* lens;
    const int32_t* cu;  // NULL: one query per sequence
    const int64_t* mask;
    int words;
    int S, T, max_tree, Hq, Hkv, G;
    float scale;
    char* out;
    int64_t ot, oh;
    float* ws;  // [T][Hq][P][D + 2]: acc[0:D], max, sum
    int P;      // partitions per sequence in the grid and the workspace
    int part;   // keys per partition
    int32_t* status;
};

// One sequence as every CTA of it sees it.
struct TreeSeq {
    int q0, n;    // first query row, query tokens (at most max_tree)
    int ctx, L;   // context keys, keys in all
    int nparts;   // partitions with keys (at least 1)
};

__device__ __forceinline__ TreeSeq tree_seq(const TreeDev& a, int s) {
    TreeSeq w;
    int ctx = __ldg(a.lens + s), bad = 0;
    if (ctx < 0) {
        ctx = 0;
        bad = QF_FLAG_BAD_TABLE;
    }
    int keys_n = 0;  // drafted keys
    if (a.cu) {
        const int b = __ldg(a.cu + s), e = __ldg(a.cu + s + 1);
        const int q0 = min(max(b, 0), a.T), q1 = min(max(e, q0), a.T);
        if (q0 != b || q1 != e) bad |= QF_FLAG_BAD_TABLE;
        w.q0 = q0;
        keys_n = q1 - q0;
        w.n = min(keys_n, a.max_tree);
        if (w.n < keys_n) bad |= QF_FLAG_BAD_TREE;
        keys_n = w.n;
    } else {
        w.q0 = s;
        w.n = 1;
    }
    if (ctx > a.cap - keys_n) {  // (cap >= 0, keys_n >= 0: no overflow)
        bad |= QF_FLAG_BAD_TABLE;
        ctx = min(ctx, a.cap);
    }
    w.ctx = ctx;
    w.L = min(ctx + keys_n, a.cap);
    w.nparts = max(1, (w.L + a.part - 1) / a.part);
    if (bad && threadIdx.x == 0) flag(a.status, bad);
    return w;
}

// Element offset of key j's row of kv head g in the caches; and of its scale.
// False (flagged) when its block is outside the cache.
__device__ __forceinline__ bool key_place(const TreeDev& a, const int32_t* bt, int g, int j,
                                          int64_t& row, int64_t& srow) {
    const int lb = a.B.div(j);
    const int64_t blk = __ldg(bt + lb);
    if (blk < 0 || blk >= a.N) {
        flag(a.status, QF_FLAG_BAD_BLOCK);
        return false;
    }
    const int slot = j - lb * a.B.d;
    row = blk * a.c0 + (int64_t)g * a.c1 + (int64_t)slot * a.c2;
    srow = blk * a.s0 + (int64_t)g * a.s1 + (int64_t)slot * a.s2;
    return true;
}

// Bits [i0, i0 + 32) of a query's mask row as drafted keys; keys before the
// tree (i0 < 0) are context, seen by every query.
__device__ __forceinline__ uint32_t tree_bits32(const int64_t* row, int words, int i0) {
    if (i0 <= -32) return 0xffffffffu;
    auto word = [&](int w) -> uint64_t {
        return w < words ? (uint64_t)__ldg(reinterpret_cast<const long long*>(row + w)) : 0ull;
    };
    if (i0 < 0) return ((1u << -i0) - 1u) | ((uint32_t)word(0) << -i0);
    const int w = i0 >> 6, b = i0 & 63;
    uint64_t v = word(w) >> b;
    if (b > 32) v |= word(w + 1) << (64 - b);
    return (uint32_t)v;
}

// Zero the rows of kv head g's query heads that no kernel computes: query
// tokens of this sequence past max_tree, and, from the first and the last
// sequence, the rows before and behind all sequences.
template <typename T, int D>
__device__ __forceinline__ void zero_unowned_rows(const TreeDev& a, int s, int g, const TreeSeq& w) {
    if (!a.cu) return;
    auto zero = [&](int t0, int t1) {
        constexpr int CH = D * (int)sizeof(T) / 16;
        const int64_t n = (int64_t)max(0, t1 - t0) * a.G * CH;
        for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
            const int64_t r = i / CH;
            const int c = (int)(i - r * CH), h = (int)(r % a.G);
            T* o = reinterpret_cast<T*>(a.out) + (t0 + r / a.G) * a.ot + (int64_t)(g * a.G + h) * a.oh;
            for (int e = 0; e < 16 / (int)sizeof(T); ++e)
                o[c * (16 / (int)sizeof(T)) + e] = Dt<T>::from_f(0.f);
        }
    };
    const int b = min(max(__ldg(a.cu + s), 0), a.T), e = min(max(__ldg(a.cu + s + 1), b), a.T);
    zero(b + w.n, e);
    if (s == 0) zero(0, b);
    if (s == a.S - 1) zero(e, a.T);
}

// Let a kernel take `bytes` of dynamic shared memory, once per device.
template <auto Kernel>
int allow_smem(int bytes) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return launch_failed(e);
    if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev) & 1) return QF_OK;
    e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return launch_failed(e);
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return QF_OK;
}

// The 16-bit kernels: paged_tree_mma.cu for few rows per kv head (`rows` in the
// longest tree), paged_tree_tc.cu for many at head_dim 128 (`tiles` of 128 per CTA).
int launch_tree_mma(const TreeDev& a, int dtype, int format, int D, int rows, cudaStream_t stream);
int launch_tree_tc(const TreeDev& a, int dtype, int format, int tiles, cudaStream_t stream);

}  // namespace qf
