// Attention of several new tokens per sequence over the paged cache (a tree of
// drafted tokens), and decode over a quantised cache: entry points, the fp32
// kernel, the merge of split sequences, and the trees' visibility masks.
//
//   out[t, h] = softmax(q[t, h] . K^T * scale over the keys t sees) @ V
// in one pass over the keys with a running maximum m and sum l per row
// (scores in units of log2, so exp is 2^x).  The rows of one kv head are its
// G = Hq / Hkv query heads of every query token, r = token * G + head: they all
// read the same K and V, so a sequence's cache crosses HBM once per row tile.
//
// Which kernel:
//  * float32: the CUDA-core kernel here (any cache format);
//  * 16-bit, up to kMmaRows rows (codes: kMmaRows8), or head_dim 64 / 256: paged_tree_mma.cu
//    (mma.sync, operands straight from global memory);
//  * 16-bit, head_dim 128, more rows: paged_tree_tc.cu (tcgen05).
#include <math.h>

#include "qf_mma.cuh"
#include "qf_quant.cuh"
#include "qf_tree.cuh"

namespace qf {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
// Rows per kv head that the mma.sync kernel takes at head_dim 128, over 16-bit and over
// 8-bit rows (it reads the cache once per 16 of them, the tcgen05 kernel once per 256).
// 32 trees at 4096 context keys, 8 kv heads, pages of 16, mma.sync | tcgen05: bf16, 8 rows
// 101 | 106 us, 16 rows 101 | 106, 24 rows 182 | 107; e4m3, 16 rows 85 | 171, 24 rows 148 |
// 170, 32 rows 154 | 156 (int8 167 | 144), 48 rows 220 | 176; 2 trees at 700 keys, bf16, 16
// rows 13.9 | 16.4, 24 rows 16.9 | 16.4.  The same with 2 kv heads and pages of 64: bf16, 16
// rows 40.8 | 41.9, 24 rows 57.0 | 42.2; e4m3, 24 rows 48.1 | 58.0, 32 rows 49.5 | 56.8.
constexpr int kMmaRows = 16, kMmaRows8 = 24;
constexpr int kF32Keys = 64;  // keys of a work unit of the fp32 kernel

// ---------------------------------------------------------------------------
// fp32.  A CTA of 4 warps takes NR = 4 WR rows and steps through tiles of 32
// keys in shared memory, as floats (codes are decoded on the way in).  WR warps
// divide the rows, 4 / WR the keys of a tile: 4 x 1 for many rows, 1 x 4 for a
// decode step's few.  QK: a lane owns one key and 4 rows (or 1 of each),
// reading K by 16 bytes from rows padded to D + 4 floats and q as a broadcast;
// PV: a lane owns D / 32 output columns.  Bound by shared-memory reads (5
// 16-byte reads for 16 multiply-adds a lane): 8 trees of 16 nodes x 4 heads at 4096
// keys, 8 kv heads of 128, in 627 us (14 TFLOP/s); decode of 32 sequences x 4 heads over
// e4m3 at 4096 keys in 342 us.
template <int FMT, int D, int WR>
struct F32Tile {
    static constexpr int WK = 4 / WR, NR = 4 * WR, KW = 32 / WK, KROW = D + 4;
    static constexpr int Q = NR * D, K = 32 * KROW, V = 32 * D, PS = 4 * 4 * KW;
    static constexpr int FLOATS = Q + K + V + PS + 4 * 4 + 32;
    static_assert(WK * NR * D + 2 * WK * NR <= K + V, "merge area");
};

// 16 bytes' worth of a cache row as floats: 4 fp32 elements or 16 codes.
template <int FMT>
__device__ __forceinline__ void decode16(const uint4& v, float scale, float* f) {
    if constexpr (FMT == QF_CACHE_PLAIN) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(word(v, i));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) codes_to_float<FMT>(word(v, i), f + 4 * i);
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] *= scale;
    }
}

template <int FMT, int D, int WR>
__global__ void __launch_bounds__(128) tree_f32_kernel(const TreeDev a) {
    using FT = F32Tile<FMT, D, WR>;
    constexpr int WK = FT::WK, NR = FT::NR, KW = FT::KW, KROW = FT::KROW, PER = D / 32;
    constexpr int EB = FMT == QF_CACHE_PLAIN ? 4 : 1, EPC = 16 / EB;
    extern __shared__ __align__(16) float fsm[];
    float* qs = fsm;
    float* kt = qs + FT::Q;
    float* vt = kt + FT::K;
    float* ps = vt + FT::V;     // [4 warps][4 rows][KW]
    float* corr = ps + FT::PS;  // [4 warps][4 rows]
    int* kval = reinterpret_cast<int*>(corr + 16);

    __shared__ int scratch[34];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int wr = warp % WR, wk = warp / WR;
    pdl_wait();
    pdl_trigger();
    TreeWalk<kF32Keys, NR, 4> walk;
    walk.begin(a, scratch);
    zero_unowned_rows<float, D>(a);
    if (tid == 0) walk.record(a);
    TreeSeg sg;
    while (walk.next(a, sg)) {
    const TreeSeq& w = sg.w;
    const int rows = w.n * a.G, r0 = sg.rg * NR, g = sg.g, k_begin = sg.k_begin, k_end = sg.k_end;
    for (int i = tid; i < NR * D; i += 128) {
        const int r = r0 + i / D, d = i % D;
        qs[i] = r < rows ? reinterpret_cast<const float*>(a.q)[(int64_t)(w.q0 + r / a.G) * a.qt +
                                                               (int64_t)(g * a.G + r % a.G) * a.qh + d]
                         : 0.f;
    }
    const int32_t* bt = a.bt + (int64_t)sg.s * a.bts;
    const float sl2 = a.scale * kLog2e;
    constexpr int NS = 4 * KW / 32;  // scores per lane
    float m[NS], l[NS], acc[4][PER];
#pragma unroll
    for (int i = 0; i < NS; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[i][e] = 0.f;

    for (int j0 = k_begin; j0 < k_end; j0 += 32) {
        __syncthreads();  // the tile before this one has been read
        {
            const int kk = tid >> 2, part = tid & 3, j = j0 + kk;
            int64_t row = 0, srow = 0;
            const bool ok = j < k_end && key_place(a, bt, g, j, row, srow);
            float ksc = 1.f, vsc = 1.f;
            if (FMT != QF_CACHE_PLAIN && ok) {
                ksc = __ldg(a.ks + srow);
                vsc = __ldg(a.vs + srow);
            }
            if (part == 0) kval[kk] = ok;
#pragma unroll
            for (int c = part; c < D / EPC; c += 4) {
                float f[EPC];
                const uint4 z = make_uint4(0, 0, 0, 0);
                decode16<FMT>(ok ? ld_shared_ro16(a.kc + (row + c * EPC) * EB) : z, ksc, f);
#pragma unroll
                for (int e = 0; e < EPC; e += 4)
                    *reinterpret_cast<float4*>(kt + kk * KROW + c * EPC + e) =
                        make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
                decode16<FMT>(ok ? ld_shared_ro16(a.vc + (row + c * EPC) * EB) : z, vsc, f);
#pragma unroll
                for (int e = 0; e < EPC; e += 4)
                    *reinterpret_cast<float4*>(vt + kk * D + c * EPC + e) =
                        make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
            }
        }
        __syncthreads();
        const bool draft = a.cu && j0 + 32 > w.ctx;
        const int key = wk * KW + (NS == 4 ? lane : lane % KW);
        float sc[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) sc[i] = 0.f;
        const int row0 = wr * 4 + (NS == 4 ? 0 : lane / KW);  // this lane's first row in the CTA
        const float* kr = kt + key * KROW;
#pragma unroll 4
        for (int d = 0; d < D; d += 4) {
            const float4 kv = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const float4 qv = *reinterpret_cast<const float4*>(qs + (row0 + i) * D + d);
                sc[i] = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, fmaf(qv.z, kv.z, fmaf(qv.w, kv.w, sc[i]))));
            }
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int r = r0 + row0 + i;
            bool sees = kval[key] && r < rows;
            if (draft && sees)
                sees = (tree_bits32(a.mask + (int64_t)(w.q0 + r / a.G) * a.words, a.words,
                                    j0 - w.ctx) >> key) & 1;
            const float t = sees ? sc[i] * sl2 : -INFINITY;
            float mx = t;
#pragma unroll
            for (int o = KW / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.f : mn;
            const float c = exp2f(m[i] - base);
            const float pr = exp2f(t - base);
            m[i] = mn;
            l[i] = l[i] * c + pr;  // this lane's part of the row's sum
            const int ri = NS == 4 ? i : lane / KW;
            ps[(warp * 4 + ri) * KW + (NS == 4 ? lane : lane % KW)] = sees ? pr : -1.f;
            if ((NS == 4 ? lane : lane % KW) == 0) corr[warp * 4 + ri] = c;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float c = corr[warp * 4 + i];
#pragma unroll
            for (int e = 0; e < PER; ++e) acc[i][e] *= c;
        }
        // A key that a row does not see carries p = -1 and is left out of the
        // row: 0 times an infinity or a NaN in its V would not be 0.  (A key
        // with no place has zeros for V; rows past the last are never stored.)
        for (int kk = 0; kk < KW; ++kk) {
            float v[PER];
#pragma unroll
            for (int e = 0; e < PER; ++e)
                v[e] = vt[(wk * KW + kk) * D + (PER == 2 ? lane * 2 + e : (e / 4) * 128 + lane * 4 + e % 4)];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float pr = ps[(warp * 4 + i) * KW + kk];
                if (pr >= 0.f || isnan(pr)) {
#pragma unroll
                    for (int e = 0; e < PER; ++e) acc[i][e] = fmaf(pr, v[e], acc[i][e]);
                }
            }
        }
        __syncwarp();
    }
    // rows' sums over the lanes of a row, then the warps that share rows
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int o = KW / 2; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
    __syncthreads();
    float* wacc = kt;  // [WK][NR][D], then max and sum [WK][NR]
    float* wm = wacc + WK * NR * D;
    float* wl = wm + WK * NR;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int ri = wr * 4 + (NS == 4 ? i : lane / KW);
        if ((NS == 4 ? lane : lane % KW) == 0) {
            wm[wk * NR + ri] = m[i];
            wl[wk * NR + ri] = l[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < PER; ++e)
            wacc[(wk * NR + wr * 4 + i) * D +
                 (PER == 2 ? lane * 2 + e : (e / 4) * 128 + lane * 4 + e % 4)] = acc[i][e];
    __syncthreads();
    for (int i = tid; i < NR * D; i += 128) {
        const int ri = i / D, d = i % D, r = r0 + ri;
        if (r >= rows) break;
        float M = -INFINITY, Ls = 0.f, A = 0.f;
#pragma unroll
        for (int k = 0; k < WK; ++k) M = fmaxf(M, wm[k * NR + ri]);
#pragma unroll
        for (int k = 0; k < WK; ++k) {
            const float f = M == -INFINITY ? 0.f : exp2f(wm[k * NR + ri] - M);
            Ls += wl[k * NR + ri] * f;
            A += wacc[(k * NR + ri) * D + d] * f;
        }
        const int64_t t = w.q0 + r / a.G, h = g * a.G + r % a.G;
        if (sg.slot < 0) {
            reinterpret_cast<float*>(a.out)[t * a.ot + h * a.oh + d] = Ls == 0.f ? 0.f : A / Ls;
        } else {
            float* o = tree_partial(a, gridDim.x, blockIdx.x, sg.slot, NR, ri, D);
            o[d] = A;
            if (d == 0) {
                o[D] = M;
                o[D + 1] = Ls;
            }
        }
    }
    __syncthreads();  // the merge area becomes the tiles again
    }
}

template <int FMT, int D, int WR>
int launch_f32(const TreeDev& a, int ctas, cudaStream_t stream) {
    constexpr auto kernel = tree_f32_kernel<FMT, D, WR>;
    constexpr int smem = F32Tile<FMT, D, WR>::FLOATS * 4;
    const int rc = allow_smem<kernel>(smem);
    if (rc) return rc;
    return launch_pdl(kernel, dim3((unsigned)ctas), 128, (size_t)smem, stream, a);
}

template <int FMT, int D>
int launch_f32(const TreeDev& a, int rows, int ctas, cudaStream_t stream) {
    return rows == 4 ? launch_f32<FMT, D, 1>(a, ctas, stream) : launch_f32<FMT, D, 4>(a, ctas, stream);
}

template <int FMT>
int launch_f32(const TreeDev& a, int D, int rows, int ctas, cudaStream_t stream) {
    switch (D) {
    case 64: return launch_f32<FMT, 64>(a, rows, ctas, stream);
    case 128: return launch_f32<FMT, 128>(a, rows, ctas, stream);
    default: return launch_f32<FMT, 256>(a, rows, ctas, stream);
    }
}

// ---------------------------------------------------------------------------
// Join the partials of the items that a CTA began and later ones went on with:
// blockIdx.x + 1 is the item's second CTA, whose record has it.  A row's partials (acc[D],
// reference in log2 units, sum) are read by one warp where they are few, two in flight, so
// that many rows are under way at once; else by eight, eight each in flight.  Bound by the
// latency of three dependent reads.  SPREAD: a CTA per row, for few items of many CTAs
// each (decode of one sequence of 131071 keys x 8 heads of 8 rows: 71 us, else 96; of 4 of
// 4000 keys 17 | 22); else a CTA for eight rows (32 trees of 4 nodes x 4 heads at 4096
// keys over e4m3: 84 us, a CTA a row 95).
template <typename T, int D>
struct Join {
    static constexpr int PER = D / 32;  // columns per lane
    float part[8][D], tops[8], sums[8];

    // Row r of the item, by WPR warps, this one the sub-th: n partials, the first of them
    // CTA `first`'s second, the others the first ones of the CTAs behind it.
    template <int WPR>
    __device__ __forceinline__ void row(const TreeDev& a, const TreeRec& rec, int64_t ctas, int64_t first, int n,
                                        int rows_per_item, int ri, int sub) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        auto partial = [&](int p) -> const float* {
            return tree_partial(a, ctas, first + p, p == 0 ? 1 : 0, rows_per_item, ri, D);
        };
        // this warp's partials against their own largest reference
        float M = -INFINITY, Ls = 0.f, acc[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] = 0.f;
        for (int p = sub + WPR * lane; p < n; p += WPR * 32) M = fmaxf(M, partial(p)[D]);
        M = warp_max(M);
        const float base = M == -INFINITY ? 0.f : M;
#pragma unroll (WPR == 1 ? 2 : 8)
        for (int p = sub; p < n; p += WPR) {
            const float* wp = partial(p);
            const float2 ml = *reinterpret_cast<const float2*>(wp + D);
            // (a factor in two halves: a sum may be 2^100 and more where V's scales are in
            // the reference)
            const float h = exp2f(0.5f * (ml.x - base)), f = h * h;
            Ls += ml.y * h * h;
#pragma unroll
            for (int e = 0; e < PER; e += 2) {
                const float2 v = *reinterpret_cast<const float2*>(wp + e * 32 + lane * 2);
                acc[e] += v.x * f;
                acc[e + 1] += v.y * f;
            }
        }
#pragma unroll
        for (int e = 0; e < PER; e += 2)
            *reinterpret_cast<float2*>(&part[warp][e * 32 + lane * 2]) = make_float2(acc[e], acc[e + 1]);
        if (lane == 0) tops[warp] = M, sums[warp] = Ls;
        if (WPR > 1) __syncthreads();
        else __syncwarp();
        // the row's warps share its columns
        const int w0 = warp - sub, r = rec.r0 + ri, tok = r / a.G;
        T* o = reinterpret_cast<T*>(a.out) + (int64_t)(rec.q0 + tok) * a.ot +
               (int64_t)(rec.g * a.G + r - tok * a.G) * a.oh;
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < WPR; ++k) top = fmaxf(top, tops[w0 + k]);
        float f[WPR], total = 0.f;
#pragma unroll
        for (int k = 0; k < WPR; ++k) {
            const float h = top == -INFINITY ? 0.f : exp2f(0.5f * (tops[w0 + k] - top));
            f[k] = h * h;
            total += sums[w0 + k] * h * h;
        }
        for (int d = sub * 32 + lane; d < D; d += WPR * 32) {
            float A = 0.f;
#pragma unroll
            for (int k = 0; k < WPR; ++k) A += part[w0 + k][d] * f[k];
            // (no weight at all: 0, or NaN where every key the row sees has a NaN for a scale)
            o[d] = Dt<T>::from_f(total == 0.f ? A * 0.f : A / total);
        }
    }
};

template <typename T, int D, bool SPREAD>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeDev a, int rows_per_item) {
    constexpr int RPC = SPREAD ? 1 : 8;  // rows per CTA
    __shared__ __align__(8) Join<T, D> join;
    pdl_wait();
    const int warp = threadIdx.x >> 5;
    const int64_t ctas = gridDim.x + 1, cta = blockIdx.x + 1;
    const TreeRec rec = reinterpret_cast<const TreeRec*>(a.ws)[cta];
    const int ri = blockIdx.y * RPC, rows = min(rows_per_item, rec.rows - rec.r0);
    if (rec.last == 0 || ri >= rows) return;
    const int n = rec.last - (int)cta + 2;
    if (!SPREAD && n <= 8) {
        if (ri + warp < rows) join.template row<1>(a, rec, ctas, cta - 1, n, rows_per_item, ri + warp, 0);
        return;
    }
    for (int i = ri; i < min(ri + RPC, rows); ++i) {
        join.template row<8>(a, rec, ctas, cta - 1, n, rows_per_item, i, warp);
        if (RPC > 1) __syncthreads();
    }
}

template <typename T, int D>
int launch_merge(const TreeDev& a, int rows, int ctas, bool spread, cudaStream_t stream) {
    if (spread)
        return launch_pdl(tree_merge_kernel<T, D, true>, dim3((unsigned)ctas - 1, (unsigned)rows), 256, 0, stream,
                          a, rows);
    return launch_pdl(tree_merge_kernel<T, D, false>, dim3((unsigned)ctas - 1, (unsigned)(rows + 7) / 8), 256, 0,
                      stream, a, rows);
}

template <typename T>
int launch_merge(const TreeDev& a, int D, int rows, int ctas, bool spread, cudaStream_t stream) {
    switch (D) {
    case 64: return launch_merge<T, 64>(a, rows, ctas, spread, stream);
    case 128: return launch_merge<T, 128>(a, rows, ctas, spread, stream);
    default: return launch_merge<T, 256>(a, rows, ctas, spread, stream);
    }
}

// ---------------------------------------------------------------------------
// A CTA per sequence, a thread per node: walk from the node to its root.  The
// walk's indices only fall, so the mask's words come out from the last to the
// first, each once.  Latency-bound: depth dependent reads, which the first
// level cache answers; 256 trees of up to 127 nodes in 5.3 us.
__global__ void __launch_bounds__(128)
    build_tree_mask_kernel(const void* parents, int index_type, const int32_t* cu, int S, int T,
                           int max_tree, int words, int64_t* mask, int32_t* depths, int32_t* status) {
    pdl_wait();
    pdl_trigger();
    const int s = blockIdx.x;
    const int b = min(max(__ldg(cu + s), 0), T), e = min(max(__ldg(cu + s + 1), b), T);
    auto empty = [&](int t0, int t1) {
        for (int t = t0 + (int)threadIdx.x; t < t1; t += blockDim.x) {
            for (int i = 0; i < words; ++i) mask[(int64_t)t * words + i] = 0;
            depths[t] = 0;
        }
    };
    if (s == 0) empty(0, b);
    if (s == S - 1) empty(e, T);
    if (e - b > max_tree) {
        if (threadIdx.x == 0) flag(status, QF_FLAG_BAD_TREE);
        empty(b + max_tree, e);
    }
    for (int i = threadIdx.x; i < min(e - b, max_tree); i += blockDim.x) {
        int64_t* row = mask + (int64_t)(b + i) * words;
        int node = i, depth = -1, word = words - 1;
        uint64_t bits = 0;
        while (node >= 0) {
            for (; word > (node >> 6); --word) {
                row[word] = (int64_t)bits;
                bits = 0;
            }
            bits |= 1ull << (node & 63);
            ++depth;
            const int64_t up = load_index(parents, (int64_t)b + node, index_type);
            if (up < -1 || up >= node) {
                flag(status, QF_FLAG_BAD_TREE);
                node = -1;
            } else {
                node = (int)up;
            }
        }
        for (; word >= 0; --word) {
            row[word] = (int64_t)bits;
            bits = 0;
        }
        depths[b + i] = depth;
    }
}

// ---------------------------------------------------------------------------
struct TreePlan {
    int tiles;      // row tiles per CTA of the tcgen05 kernel; 0: another kernel
    int rows;       // rows per work item
    int ctas;       // persistent CTAs: as many as fit, or one per unit of work if that is fewer
    bool split;     // whether sequences may be cut
    bool spread;    // whether joining an item's rows is for a CTA each (see tree_merge_kernel)
    bool fits;      // whether the work has fewer than 2^31 units
};

// The kernel and its grid, by sizes alone (lengths are on the device; the block
// tables bound them).  A cut costs a partial of (D + 2) floats a row, written and
// read back, so a CTA's stretch is at least two blocks of keys; and a second launch, so
// sequences of up to 768 keys (256 of the mma.sync kernel's) stay whole.  Whole | cut: a
// tree of 16 nodes x 4 heads, 8 kv heads, at 500 keys 15.3 | 16.9 us, at 1000 18.3 |
// 17.1, at 2000 26.7 | 18.7; 8 of them at 500 keys 16.4 | 22.9; decode of 4 sequences
// over e4m3 at 200 keys 8.6 | 9.2 us, at 500 13.1 | 10.6, at 1000 23.7 | 11.9.
TreePlan make_plan(const qf_paged_tree_attention_args& g) {
    TreePlan p{};
    const int64_t G = g.num_q_heads / g.num_kv_heads, rows = (g.cu_seqlens_q ? g.max_tree : 1) * G;
    int64_t per_sm, keys = 64;
    const bool plain = g.cache_format == QF_CACHE_PLAIN;
    if (g.dtype == QF_F32) {
        p.rows = rows <= 4 ? 4 : 16;
        per_sm = g.head_dim == 256 ? 2 : 4;
    } else if (g.head_dim == 128 && rows > (plain ? kMmaRows : kMmaRows8)) {
        p.tiles = rows > 128 ? 2 : 1;
        p.rows = 128 * p.tiles;
        per_sm = 1;
        keys = 128;
    } else {
        p.rows = g.head_dim == 256 || rows <= 8 ? 8 : 16;
        per_sm = tree_mma_ctas_per_sm(plain, (int)g.head_dim);
    }
    const int64_t cap = std::max<int64_t>(1, g.max_blocks_per_seq * g.block_size);
    const int64_t blocks = ceil_div(cap, keys);  // of the longest sequence
    const int64_t items = g.num_seqs * g.num_kv_heads * ceil_div(rows, p.rows);
    const int64_t slots = (int64_t)sm_count() * per_sm;
    p.split = blocks > (keys == 128 ? 6 : 4);
    p.ctas = (int)(items >= slots ? slots : std::min(slots, items * blocks));
    p.spread = p.rows <= 16 && p.ctas >= 4 * items;
    p.fits = items <= INT32_MAX / (blocks + 8);
    return p;
}

bool known_sizes(const qf_paged_tree_attention_args& g) {
    return g.num_seqs > 0 && g.num_tokens > 0 && g.num_q_heads > 0 && g.num_kv_heads > 0 &&
           g.head_dim > 0 && g.block_size > 0 && g.max_blocks_per_seq >= 0 && g.max_tree >= 0 &&
           g.num_q_heads % g.num_kv_heads == 0 && g.block_size <= (1 << 30) &&
           g.max_blocks_per_seq <= (1 << 30) / g.block_size;
}

int check_tree_args(const qf_paged_tree_attention_args& g) {
    if (g.num_seqs < 0 || g.num_tokens < 0 || g.num_q_heads <= 0 || g.num_kv_heads <= 0 ||
        g.block_size <= 0 || g.num_blocks < 0 || g.max_blocks_per_seq < 0 || g.max_tree < 0 ||
        g.mask_words < 0)
        return QF_ERR_INVALID;
    if (g.num_q_heads % g.num_kv_heads) return QF_ERR_INVALID;
    if (g.dtype != QF_F32 && g.dtype != QF_F16 && g.dtype != QF_BF16) return QF_ERR_INVALID;
    if (g.cache_format != QF_CACHE_PLAIN && g.cache_format != QF_CACHE_E4M3 &&
        g.cache_format != QF_CACHE_INT8)
        return QF_ERR_INVALID;
    if (g.head_dim != 64 && g.head_dim != 128 && g.head_dim != 256) return QF_ERR_UNSUPPORTED;
    if (g.num_tokens == 0) return QF_OK;
    if (g.num_seqs == 0) return QF_ERR_INVALID;  // rows that no sequence owns
    if (!g.q || !g.k_cache || !g.v_cache || !g.context_lens || !g.out ||
        (g.max_blocks_per_seq > 0 && !g.block_tables))
        return QF_ERR_INVALID;
    if (g.cu_seqlens_q) {
        if (g.max_tree < 1 || !g.tree_mask || g.mask_words < 1) return QF_ERR_INVALID;
        if (g.mask_words < g.max_tree / 64 + (g.max_tree % 64 != 0)) return QF_ERR_INVALID;
    } else if (g.num_tokens != g.num_seqs) {
        return QF_ERR_INVALID;
    }
    if (g.cache_format != QF_CACHE_PLAIN && (!g.k_scale || !g.v_scale)) return QF_ERR_INVALID;
    if (!known_sizes(g) || g.num_seqs > 65535 || g.num_kv_heads > 65535 || g.max_tree > 65535 ||
        g.mask_words > INT32_MAX || g.num_tokens > INT32_MAX || g.num_q_heads > (1 << 20))
        return QF_ERR_UNSUPPORTED;
    const int64_t es = g.dtype == QF_F32 ? 4 : 2, cs = g.cache_format == QF_CACHE_PLAIN ? es : 1;
    // rows of q, of out and of the caches are read and written in 16-byte chunks
    if ((g.q_stride_token * es) % 16 || (g.q_stride_head * es) % 16 || !aligned16(g.q) ||
        (g.cache_strides[0] * cs) % 16 || (g.cache_strides[1] * cs) % 16 ||
        (g.cache_strides[2] * cs) % 16 || g.cache_strides[3] != 1 || !aligned16(g.k_cache) ||
        !aligned16(g.v_cache) || !aligned16(g.workspace) || (g.out_stride_token * es) % 16 ||
        (g.out_stride_head * es) % 16 || !aligned16(g.out))
        return QF_ERR_UNSUPPORTED;
    return QF_OK;
}

size_t plan_bytes(const qf_paged_tree_attention_args& g, const TreePlan& p) {
    if (!p.split || p.ctas < 2) return 0;
    return (size_t)TreeWs::floats(p.ctas, p.rows, g.head_dim) * sizeof(float);
}

int launch_tree_f32(const TreeDev& a, int format, int D, int rows, int ctas, cudaStream_t stream) {
    switch (format) {
    case QF_CACHE_PLAIN: return launch_f32<QF_CACHE_PLAIN>(a, D, rows, ctas, stream);
    case QF_CACHE_E4M3: return launch_f32<QF_CACHE_E4M3>(a, D, rows, ctas, stream);
    default: return launch_f32<QF_CACHE_INT8>(a, D, rows, ctas, stream);
    }
}

}  // namespace
}  // namespace qf

extern "C" size_t qf_paged_tree_attention_workspace_bytes(const qf_paged_tree_attention_args* p) {
    if (!p || !qf::known_sizes(*p)) return 0;
    qf_paged_tree_attention_args g = *p;
    size_t bytes = qf::plan_bytes(g, qf::make_plan(g));
    if (!g.cu_seqlens_q) {
        static const int32_t some = 0;
        g.cu_seqlens_q = &some;  // (whether there is one is all that is read)
        bytes = std::max(bytes, qf::plan_bytes(g, qf::make_plan(g)));
    }
    return bytes;
}

extern "C" size_t qf_paged_tree_attention_args_size(void) {
    return sizeof(qf_paged_tree_attention_args);
}

extern "C" int qf_paged_tree_attention(const qf_paged_tree_attention_args* p, cudaStream_t stream) {
    if (!p) return QF_ERR_INVALID;
    const qf_paged_tree_attention_args& g = *p;
    int rc = qf::check_tree_args(g);
    if (rc || g.num_tokens == 0) return rc;
    const qf::TreePlan plan = qf::make_plan(g);
    if (!plan.fits) return QF_ERR_UNSUPPORTED;
    const size_t need = qf::plan_bytes(g, plan);
    if (need > 0 && g.workspace) {
        if (g.workspace_bytes < 0 || (size_t)g.workspace_bytes < need) return QF_ERR_INVALID;
    }
    qf::TreeDev a{};
    a.q = static_cast<const char*>(g.q);
    a.qt = g.q_stride_token;
    a.qh = g.q_stride_head;
    a.kc = static_cast<const char*>(g.k_cache);
    a.vc = static_cast<const char*>(g.v_cache);
    a.c0 = g.cache_strides[0];
    a.c1 = g.cache_strides[1];
    a.c2 = g.cache_strides[2];
    a.ks = g.k_scale;
    a.vs = g.v_scale;
    a.s0 = g.scale_strides[0];
    a.s1 = g.scale_strides[1];
    a.s2 = g.scale_strides[2];
    a.N = g.num_blocks;
    a.B = qf::FastDiv((int)g.block_size);
    a.bt = g.block_tables;
    a.bts = g.block_tables_row_stride;
    a.cap = (int)(g.max_blocks_per_seq * g.block_size);
    a.lens = g.context_lens;
    a.cu = g.cu_seqlens_q;
    a.mask = g.tree_mask;
    a.words = (int)g.mask_words;
    a.S = (int)g.num_seqs;
    a.T = (int)g.num_tokens;
    a.max_tree = g.cu_seqlens_q ? (int)g.max_tree : 1;
    a.Hq = (int)g.num_q_heads;
    a.Hkv = (int)g.num_kv_heads;
    a.G = a.Hq / a.Hkv;
    a.scale = g.scale;
    a.out = static_cast<char*>(g.out);
    a.ot = g.out_stride_token;
    a.oh = g.out_stride_head;
    a.ws = need > 0 ? static_cast<float*>(g.workspace) : nullptr;
    a.status = g.status;
    const int D = (int)g.head_dim;
    if (g.dtype == QF_F32)
        rc = qf::launch_tree_f32(a, g.cache_format, D, plan.rows, plan.ctas, stream);
    else if (plan.tiles)
        rc = qf::launch_tree_tc(a, g.dtype, g.cache_format, plan.tiles, plan.ctas, stream);
    else
        rc = qf::launch_tree_mma(a, g.dtype, g.cache_format, D, plan.rows, plan.ctas, stream);
    if (rc || !a.ws) return rc;
    switch (g.dtype) {
    case QF_F32: return qf::launch_merge<float>(a, D, plan.rows, plan.ctas, plan.spread, stream);
    case QF_F16: return qf::launch_merge<__half>(a, D, plan.rows, plan.ctas, plan.spread, stream);
    default: return qf::launch_merge<__nv_bfloat16>(a, D, plan.rows, plan.ctas, plan.spread, stream);
    }
}

extern "C" int qf_build_tree_mask(const qf_tree_mask_args* p, cudaStream_t stream) {
    if (!p) return QF_ERR_INVALID;
    const qf_tree_mask_args& g = *p;
    if (g.num_seqs < 0 || g.num_nodes < 0 || g.max_tree < 1 || g.mask_words < 1) return QF_ERR_INVALID;
    if (g.index_type != QF_I32 && g.index_type != QF_I64) return QF_ERR_INVALID;
    if (g.mask_words < g.max_tree / 64 + (g.max_tree % 64 != 0)) return QF_ERR_INVALID;
    if (g.num_nodes == 0) return QF_OK;
    if (g.num_seqs == 0 || !g.parents || !g.cu_seqlens || !g.mask || !g.depths) return QF_ERR_INVALID;
    if (g.num_seqs > INT32_MAX || g.num_nodes > INT32_MAX || g.max_tree > INT32_MAX ||
        g.mask_words > INT32_MAX)
        return QF_ERR_UNSUPPORTED;
    return qf::launch_pdl(qf::build_tree_mask_kernel, dim3((unsigned)g.num_seqs), 128, 0, stream, g.parents,
                          g.index_type, g.cu_seqlens, (int)g.num_seqs, (int)g.num_nodes, (int)g.max_tree,
                          (int)g.mask_words, g.mask, g.depths, g.status);
}

extern "C" size_t qf_tree_mask_args_size(void) { return sizeof(qf_tree_mask_args); }
