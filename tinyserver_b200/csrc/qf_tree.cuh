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
    float* ws;     // partials and records (TreeWs), or NULL: no sequence is split
    int32_t* status;
};

// One sequence: its first query row, query tokens (at most max_tree), context
// keys, and keys in all.  `report`: this thread flags what had to be cut.
struct TreeSeq {
    int q0, n, ctx, L;
};

__device__ __forceinline__ TreeSeq tree_seq(const TreeDev& a, int s, bool report) {
    TreeSeq w;
    int ctx = __ldg(a.lens + s), bad = 0;
    if (ctx < 0) {
        ctx = 0;
        bad = QF_FLAG_BAD_TABLE;
    }
    int drafted = 0;
    if (a.cu) {
        const int b = __ldg(a.cu + s), e = __ldg(a.cu + s + 1);
        const int q0 = min(max(b, 0), a.T), q1 = min(max(e, q0), a.T);
        if (q0 != b || q1 != e) bad |= QF_FLAG_BAD_TABLE;
        w.q0 = q0;
        w.n = min(q1 - q0, a.max_tree);
        if (w.n < q1 - q0) bad |= QF_FLAG_BAD_TREE;
        drafted = w.n;
    } else {
        w.q0 = s;
        w.n = 1;
    }
    if (ctx > a.cap - drafted) {  // (cap, drafted >= 0: no overflow)
        bad |= QF_FLAG_BAD_TABLE;
        ctx = min(ctx, a.cap);
    }
    w.ctx = ctx;
    w.L = min(ctx + drafted, a.cap);
    if (bad && report) flag(a.status, bad);
    return w;
}

// ---------------------------------------------------------------------------
// Who does what.  The work is a line of units, one unit a block of KB keys for
// one tile group (ROWS rows) of one kv head of one sequence: sequence by
// sequence, in it head by head and group by group, in that the keys in order.
// gridDim.x CTAs, as many as fit on the GPU at once, take equal stretches of the
// line, so lengths may be as ragged as they like.  A stretch cuts at most
// two (sequence, head, group) items, its first and its last, so a CTA leaves at
// most two partials, in its own slots of the workspace: slot 0 for an item that an
// earlier CTA began, slot 1 for one that it begins and a later CTA goes on with.
// Its record says what slot 0 belongs to, for the kernel that joins them.
// An item begins with EXTRA units without keys, what Q and O cost in units, so that
// a stretch of many short items is no longer than one of few long ones.
// Without a workspace a CTA does whole items: those that begin in its stretch.
struct TreeRec {
    int last;     // the last CTA of slot 0's item; 0 unless the CTA before this one began it
    int q0;       // the item's sequence's first query token
    int g;        // its kv head
    int r0, rows;  // its first row, and the sequence's rows per kv head
    int unused[3];
};

struct TreeWs {  // workspace: records, then [CTA][2][ROWS][D + 2] floats: acc, reference, sum
    __host__ __device__ static int64_t rec_floats(int64_t ctas) { return (ctas * 8 + 63) / 64 * 64; }
    __host__ __device__ static int64_t floats(int64_t ctas, int64_t rows, int64_t d) {
        return rec_floats(ctas) + ctas * 2 * rows * (d + 2);
    }
};

struct TreeSeg {
    TreeSeq w;
    int s, g, rg;
    int k_begin, k_end;
    int slot;  // of the partial; -1: the item is whole
};

// A CTA's least stretch, in units: a partial costs about as much.  Decode of 4 sequences
// of 700 keys over e4m3 9.8 us (with 1: 9.8, with 4: 10.8).
constexpr int kMinUnits = 2;

template <int KB, int ROWS, int EXTRA>
struct TreeWalk {
    // (the launcher sees to it that all units are fewer than 2^31)
    int pos, end, base, us;  // this CTA's stretch; the current sequence's first unit and units
    int per;                 // units of a stretch
    int s, nb, ng;           // the current sequence, its key blocks and groups per head
                             // (an item: EXTRA + nb units)
    TreeSeq w;

    __device__ __forceinline__ static int blocks(const TreeSeq& w) { return max(1, (w.L + KB - 1) / KB); }
    __device__ __forceinline__ static int groups(const TreeDev& a, const TreeSeq& w) {
        return (w.n * a.G + ROWS - 1) / ROWS;
    }
    __device__ __forceinline__ static int units(const TreeDev& a, const TreeSeq& w) {
        return (EXTRA + blocks(w)) * groups(a, w) * a.Hkv;
    }
    __device__ __forceinline__ void enter(const TreeDev& a, int seq) {
        s = seq;
        w = tree_seq(a, s, false);
        nb = blocks(w);
        ng = groups(a, w);
        us = units(a, w);
    }

    // By all threads of the CTA (`scratch`: 34 words of shared memory): the units
    // of all sequences, this CTA's stretch, and the sequence it begins in.  CTA 0
    // reports what had to be cut.
    __device__ __forceinline__ void begin(const TreeDev& a, int* scratch) {
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
        const int nt = nw * 32;
        int before = 0, u = 0, first = 0, total = 0;
        // first: the units before sequence i0 + tid; all: of sequences [i0, i0 + nt)
        auto scan = [&](int i0, bool report) -> int {
            const int i = i0 + tid;
            u = i < a.S ? units(a, tree_seq(a, i, report)) : 0;
            int incl = u;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            if (lane == 31) scratch[warp] = incl;
            __syncthreads();
            int warps = 0, all = 0;
#pragma unroll 1
            for (int x = 0; x < nw; ++x) {
                if (x < warp) warps += scratch[x];
                all += scratch[x];
            }
            __syncthreads();
            first = before + warps + incl - u;
            return all;
        };
#pragma unroll 1
        for (int i0 = 0; i0 < a.S; i0 += nt) total += scan(i0, blockIdx.x == 0);
        const int ctas = (int)gridDim.x;
        per = max(kMinUnits, (total - 1) / ctas + 1);
        pos = (int)min((int64_t)total, (int64_t)per * blockIdx.x);
        end = total - pos > per ? pos + per : total;
        // the sequence with base <= pos < base + us (with up to nt sequences, scanned already)
#pragma unroll 1
        for (int i0 = 0; i0 < a.S && before <= pos; i0 += nt) {
            const int all = a.S <= nt ? total : scan(i0, false);
            if (first <= pos && pos < first + u) {
                scratch[32] = i0 + tid;
                scratch[33] = first;
            }
            before += all;
        }
        __syncthreads();
        if (pos < end) {
            base = scratch[33];
            enter(a, scratch[32]);
        }
        __syncthreads();
    }

    __device__ __forceinline__ bool next(const TreeDev& a, TreeSeg& t) {
        while (pos < end) {
            if (pos >= base + us) {
                base += us;
                enter(a, s + 1);
                continue;
            }
            const int rel = pos - base, item = rel / (EXTRA + nb), u0 = rel - item * (EXTRA + nb);
            const int u1 = min(EXTRA + nb, u0 + (end - pos));
            if (!a.ws && u0 > 0) {  // an item of the CTA before
                pos += EXTRA + nb - u0;
                continue;
            }
            const int b0 = max(0, u0 - EXTRA), b1 = a.ws ? max(0, u1 - EXTRA) : nb;
            pos += a.ws ? u1 - u0 : EXTRA + nb;
            if (b1 == 0) continue;  // the item's keys are the next CTA's
            t.w = w;
            t.s = s;
            t.g = item / ng;
            t.rg = item - t.g * ng;
            t.k_begin = b0 * KB;
            t.k_end = min(w.L, b1 * KB);
            t.slot = b0 > 0 ? 0 : b1 < nb ? 1 : -1;
            return true;
        }
        return false;
    }

    // By one thread, before the walk: the record of this CTA.
    __device__ __forceinline__ void record(const TreeDev& a) const {
        if (!a.ws) return;
        TreeRec r{};
        if (pos < end && pos > base) {
            const int rel = pos - base, item = rel / (EXTRA + nb), b0 = rel - item * (EXTRA + nb) - EXTRA;
            const int first = pos - b0;  // the unit of the item's first block
            if (b0 > 0 && first >= pos - per) {
                r.q0 = w.q0;
                r.g = item / ng;
                r.r0 = (item - r.g * ng) * ROWS;
                r.rows = w.n * a.G;
                r.last = (first + nb - 1) / per;
            }
        }
        reinterpret_cast<TreeRec*>(a.ws)[blockIdx.x] = r;
    }
};

__device__ __forceinline__ float* tree_partial(const TreeDev& a, int64_t ctas, int64_t cta, int slot,
                                               int rows, int row, int D) {
    return a.ws + TreeWs::rec_floats(ctas) + ((cta * 2 + slot) * rows + row) * (D + 2);
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

// Zero the output rows that no item owns, all CTAs together: before the first
// and behind the last sequence, and query tokens past max_tree.
template <typename T, int D>
__device__ __forceinline__ void zero_unowned_rows(const TreeDev& a) {
    if (!a.cu) return;
    const int chunks = a.Hq * (D * (int)sizeof(T) / 16);  // 16-byte pieces of a query token
    auto zero = [&](int t0, int t1) {
#pragma unroll 1
        for (int t = t0; t < t1; ++t)
#pragma unroll 1
            for (int i = threadIdx.x; i < chunks; i += blockDim.x) {
                const int h = i / (D * (int)sizeof(T) / 16), c = i % (D * (int)sizeof(T) / 16);
                st16(a.out + (t * a.ot + h * a.oh) * (int64_t)sizeof(T) + c * 16, make_uint4(0, 0, 0, 0));
            }
    };
    auto row = [&](int s) { return min(max(__ldg(a.cu + s), 0), a.T); };
    if (blockIdx.x == 0) zero(0, row(0));
    if (blockIdx.x == gridDim.x - 1) zero(max(row(a.S - 1), row(a.S)), a.T);
#pragma unroll 1
    for (int s = blockIdx.x; s < a.S; s += gridDim.x) {
        const int b = row(s), e = max(b, row(s + 1));
        if (e - b > a.max_tree) zero(b + a.max_tree, e);
    }
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
int tree_mma_ctas_per_sm(bool plain, int D);
int launch_tree_mma(const TreeDev& a, int dtype, int format, int D, int rows, int ctas,
                    cudaStream_t stream);
int launch_tree_tc(const TreeDev& a, int dtype, int format, int tiles, int ctas, cudaStream_t stream);

}  // namespace qf
