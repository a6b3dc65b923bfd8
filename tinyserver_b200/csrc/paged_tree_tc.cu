// Paged attention for many query rows per kv head (a tree's tokens x G), 16-bit
// queries, head_dim 128, on the 5th-generation tensor cores.
//
// A CTA takes NT tiles of 128 rows of one (sequence, kv head) and a partition of
// the keys in blocks of 128.  Both products run on tcgen05.mma with S, P and O in
// tensor memory, P over the S it came from:
//   S_t = Q_t K_j^T     Q, K in shared memory (128-byte swizzle)
//   softmax of row r by thread r of the tile's warpgroup, whose tensor-memory
//   lane the row is; P_t back over the first half of S_t
//   O_t += P_t V_j      A = P_t from tensor memory, V in shared memory
// Roles: 4 NT softmax warps, one MMA thread, two warps that bring K and two that
// bring V.  Pages may have any size and the rows any place, so rows are fetched
// one by one: 16-bit rows with cp.async, straight into the swizzled tile; 8-bit
// rows into registers and, converted to fp16 (exact), into the tile, so the next
// block's codes are in flight while this block's tile is in use.
//
// What bounds it: a block is 64 KB of 16-bit K and V, ~2900 cycles of an SM's
// share of HBM; a tile's softmax is 16384 exponentials, 1024 cycles of the MUFU,
// and its products 1024 cycles of the tensor core.  One tile (up to 128 rows):
// bound by HBM if something is always in flight, hence two CTAs per SM, each with
// one K and one V buffer that refill while the other product and the softmax run.
// Two tiles (more rows): one CTA per SM with two-deep rings; K and V meet 256 rows,
// and tile 0's softmax overlaps tile 1's products.
//
// Quantised rows: K's scale multiplies the score; V's enters the exponent,
// p' = 2^(t + log2 vs - m') in [0, 2^8], and the sum takes p' / vs, so that O / l is
// the definition whatever the scales' range.  Where that range exceeds 2^90 the sum takes
// its own exponential (p' may have underflowed where p has not).
// P is rounded to the operand type (fp16 over quantised rows, else the query's):
// half a step of the same size as the output's own.  Sums, maxima and O are fp32.
//
// Every wait is bounded: one that runs out sets QF_FLAG_TIMEOUT and the kernel
// finishes without its result.
#include <math.h>

#include <type_traits>

#include "qf_mma.cuh"
#include "qf_quant.cuh"
#include "qf_tc.cuh"
#include "qf_tree.cuh"

namespace qf {
namespace {

constexpr int kD = 128;
constexpr unsigned kFull = 0xffffffffu;
constexpr float kKeepLog2 = 8.f;    // the reference maximum moves when the row's has grown by 2^8
constexpr float kScaleRange = 90.f;  // log2 of the v-scales' ratio up to which one exponential will do

constexpr float kLeastScale = 7.52316384526264e-37f;  // 2^-120

template <int NT>
struct TreeTc {
    static constexpr int ST = NT;                   // K and V stages
    static constexpr int SOFT = 128 * NT;           // softmax threads
    static constexpr int MMA_WARP = 4 * NT, LOAD_WARP = MMA_WARP + 1;  // K, then V
    static constexpr int THREADS = SOFT + 32 + 64;
    static constexpr int SLOTS = 2 * ST;            // blocks whose scales and valid bits are kept
    static constexpr int SMEM = (NT + 2 * ST) * kTile + 1024;
    static constexpr uint32_t COLS = 256 * NT;      // tensor memory: S_t at 128 t, O_t behind them
};

template <int NT>
struct TreeBars {
    uint64_t q_full;
    uint64_t k_full[NT], v_full[NT], k_empty[NT], v_empty[NT];
    uint64_t info_full[2 * NT];  // a block's valid bits and scales
    uint64_t s_full[NT], p_full[NT], o_full, drain;
};

__device__ __forceinline__ void proxy_fence() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void cp_async16_at(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                 : "memory");
}

// Byte offset of 16-byte chunk c (0..15) of row r in a tile.
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
    return (uint32_t)((c >> 3) * kSlab + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// Infinities and NaN of 8 16-bit values set to zero; whether there were any.
template <typename T>
__device__ __forceinline__ bool zero_not_finite(uint4& v) {
    constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w = word(v, i);
        if ((w & E) == E) w &= 0xffff0000u, any = true;
        if ((w & (E << 16)) == (E << 16)) w &= 0xffffu, any = true;
        set_word(v, i, w);
    }
    return any;
}

// q . k over the 128 dims on the CUDA cores, k a cache row.
template <typename T, int FMT>
__device__ float dot_row(const T* q, const char* k) {
    float acc = 0.f;
    for (int d = 0; d < kD; ++d) {
        float x;
        if constexpr (FMT == QF_CACHE_PLAIN) x = Dt<T>::to_f(reinterpret_cast<const T*>(k)[d]);
        else x = code_to_float<FMT>(reinterpret_cast<const uint8_t*>(k)[d]);
        acc = fmaf(Dt<T>::to_f(q[d]), x, acc);
    }
    return acc;
}

// A drafted block's V held an infinity or a NaN, which went into the product as
// zero so that rows that do not see the key stay clean: the rows that do see it
// get p * v added to what they wrote (the sum is an infinity or a NaN whatever the
// finite part was).  Keys [j0, k_end), one row per thread.
template <typename T, int FMT, typename O>
__device__ __noinline__ void add_not_finite(const TreeDev& a, const int32_t* bt, int g, int ctx,
                                            const int64_t* mrow, const T* q, float sl2, float mref,
                                            int j0, int k_end, O* out) {
    for (int j = j0; j < k_end; ++j) {
        if (!((tree_bits32(mrow, a.words, j - ctx)) & 1u)) continue;
        int64_t row, srow;
        if (!key_place(a, bt, g, j, row, srow)) continue;
        float p = -1.f;
        for (int d = 0; d < kD; ++d) {
            float v;
            if constexpr (FMT == QF_CACHE_PLAIN) v = Dt<T>::to_f(reinterpret_cast<const T*>(a.vc)[row + d]);
            else v = code_to_float<FMT>(reinterpret_cast<const uint8_t*>(a.vc)[row + d]);
            if (isfinite(v)) continue;
            if (p == -1.f) {
                float t = dot_row<T, FMT>(q, a.kc + row * (FMT == QF_CACHE_PLAIN ? 2 : 1)) * sl2;
                if constexpr (FMT != QF_CACHE_PLAIN) t = t * a.ks[srow] + log2f(a.vs[srow]);
                p = exp2f(t - mref);
            }
            out[d] = Dt<O>::from_f(Dt<O>::to_f(out[d]) + p * v);
        }
    }
}

// TMA: box {64 dims, `box` slots, 1 head, 1 block} at (x, slot, head, block) into `dst`.
__device__ __forceinline__ void tma_page(void* dst, const CUtensorMap* map, int x, int slot, int head,
                                         int block, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(slot), "r"(head), "r"(block), "r"(smem_u32(bar))
        : "memory");
}

// S_t = Q_t K^T: head_dim in steps of 16.
__device__ __forceinline__ void issue_scores(uint32_t d, uint32_t q, uint32_t k, uint32_t id) {
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
        const uint32_t off = (uint32_t)((kk >> 2) * kSlab + (kk & 3) * 32);
        mma_ss(d, sdesc(q + off, 16, 1024), sdesc(k + off, 16, 1024), id, kk > 0 ? 1u : 0u);
    }
}

template <typename T, int FMT, int NT>
__global__ void __launch_bounds__(TreeTc<NT>::THREADS, NT == 1 ? 2 : 1)
    tree_tc_kernel(const TreeDev a, const __grid_constant__ CUtensorMap tk,
                   const __grid_constant__ CUtensorMap tv, int box) {
    using C = TreeTc<NT>;
    constexpr bool Q8 = FMT != QF_CACHE_PLAIN;
    using MT = typename std::conditional<Q8, __half, T>::type;
    using MP = Packed<MT>;
    constexpr int ST = C::ST;

    const int p = blockIdx.x, s = blockIdx.z;
    const int g = blockIdx.y % a.Hkv, rg = blockIdx.y / a.Hkv;
    const TreeSeq w = tree_seq(a, s);
    if (p == 0 && rg == 0) zero_unowned_rows<T, kD>(a, s, g, w);
    const int rows = w.n * a.G, r0 = rg * NT * kRows;
    if (p >= w.nparts || r0 >= rows) return;
    const int k_begin = p * a.part, k_end = k_begin + min(w.L - k_begin, a.part);
    const int nblk = (k_end - k_begin + kRows - 1) / kRows;
    const int ntile = min(NT, (rows - r0 + kRows - 1) / kRows);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // where this softmax thread's row goes
    const int trow = r0 + (tid & (NT * kRows - 1));
    const bool live = tid < C::SOFT && trow < rows;
    const int tok = live ? trow / a.G : 0;
    const int hq = g * a.G + (live ? trow - tok * a.G : 0);
    const int64_t trow_q = w.q0 + tok;
    T* const orow = reinterpret_cast<T*>(a.out) + trow_q * a.ot + (int64_t)hq * a.oh;
    if (nblk == 0) {  // no key at all
        if (live)
            for (int c = 0; c < kD / 8; ++c) st16(orow + 8 * c, make_uint4(0, 0, 0, 0));
        return;
    }

    extern __shared__ __align__(1024) char dsm[];
    __shared__ TreeBars<NT> bars;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, odd_v;
    __shared__ uint32_t valid[C::SLOTS][4];
    // k-scale, log2 v-scale, 1 / v-scale of a block's keys; least and largest log2 v-scale
    __shared__ __align__(16) float sk[Q8 ? C::SLOTS : 1][Q8 ? kRows : 1], sl[Q8 ? C::SLOTS : 1][Q8 ? kRows : 1],
        sr_[Q8 ? C::SLOTS : 1][Q8 ? kRows : 1];
    __shared__ float srange[Q8 ? C::SLOTS : 1][2];
    volatile int* abort = &abort_flag;

    const uint32_t raw = smem_u32(dsm);
    char* base = dsm + (((raw + 1023u) & ~1023u) - raw);
    char* const kbase = base + NT * kTile;
    char* const vbase = kbase + ST * kTile;
    if (tid == 0) {
        mbar_init(&bars.q_full, (uint32_t)(ntile * kRows));
        for (int i = 0; i < ST; ++i) {
            mbar_init(&bars.k_full[i], 32);
            mbar_init(&bars.v_full[i], 32);
            mbar_init(&bars.k_empty[i], 1);
            mbar_init(&bars.v_empty[i], 1);
        }
        for (int i = 0; i < C::SLOTS; ++i) mbar_init(&bars.info_full[i], 32);
        for (int t = 0; t < NT; ++t) {
            mbar_init(&bars.s_full[t], 1);
            mbar_init(&bars.p_full[t], kRows);
        }
        mbar_init(&bars.o_full, 1);
        mbar_init(&bars.drain, 1);
        abort_flag = 0;
        odd_v = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == C::MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_slot)),
                     "r"(C::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const int32_t* bt = a.bt + (int64_t)s * a.bts;
    const float sl2 = a.scale * 1.4426950408889634f;
    const bool tree = a.cu != nullptr;
    // the first block that a row may not see whole
    const int first_draft = tree ? max(0, (w.ctx - k_begin) / kRows) : nblk;

    if (warp >= C::LOAD_WARP) {
        // ---- loaders: one warp K, one warp V
        const int side = warp - C::LOAD_WARP;
        const char* src = side ? a.vc : a.kc;
        char* const tiles = side ? vbase : kbase;
        uint64_t* full = side ? bars.v_full : bars.k_full;
        uint64_t* empty = side ? bars.v_empty : bars.k_empty;
        // lane l: keys l, l + 32, l + 64, l + 96 of a block
        int64_t off[4];
        unsigned ok[4];
        float ks[4], vs[4];
        auto locate = [&](int j) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int key = k_begin + j * kRows + x * 32 + lane;
                int64_t srow = 0;
                off[x] = 0;
                ks[x] = 0.f;
                vs[x] = 1.f;
                const bool in = key < k_end && key_place(a, bt, g, key, off[x], srow);
                ok[x] = __ballot_sync(kFull, in);
                if (!Q8) off[x] *= 2;  // bytes
                if (Q8 && side == 0 && in) {
                    ks[x] = __ldg(a.ks + srow);
                    vs[x] = __ldg(a.vs + srow);
                    // a scale of 0 (a row never written) stands for zeros, as good as at 2^-120
                    if (vs[x] < kLeastScale) vs[x] = kLeastScale;
                }
            }
        };
        // What the softmax needs to know of block j's keys.  The slot's last reader, the
        // softmax of block j - SLOTS, is done: S of block j - ST (whose K was in this
        // stage) came after it.
        auto inform = [&](int slot) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                if (lane == 0) valid[slot][x] = ok[x];
                if constexpr (Q8) {
                    sk[slot][x * 32 + lane] = ks[x];
                    sl[slot][x * 32 + lane] = log2f(vs[x]);
                    sr_[slot][x * 32 + lane] = 1.f / vs[x];
                }
            }
            if constexpr (Q8) {
                float hi = -INFINITY, lo = -INFINITY;
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if ((ok[x] >> lane) & 1) {
                        hi = fmaxf(hi, log2f(vs[x]));
                        lo = fmaxf(lo, -log2f(vs[x]));
                    }
                hi = warp_max(hi);
                lo = -warp_max(lo);
                if (lane == 0) srange[slot][0] = lo, srange[slot][1] = hi;
            }
            __syncwarp();
            mbar_arrive(&bars.info_full[slot]);
        };
        // block j's stage may be refilled (the whole warp learns the same)
        auto vacant = [&](int j) -> bool {
            return __all_sync(kFull, j < ST || mbar_wait(&empty[j % ST], ((j / ST) - 1) & 1, abort));
        };
        if constexpr (Q8) {
            // codes into registers, 16 rows' worth a lane group in flight all the time: half a
            // block is converted and stored while the other half, then the next block's, comes
            uint4 raws[16];
            const int c = lane & 7;
            auto fetch = [&](int i, int half) {
                const int r = (4 * i + (lane >> 3)) & 31, x = 2 * half + (i >> 3);
                const int64_t o = __shfl_sync(kFull, x == 0 ? off[0] : x == 1 ? off[1] : x == 2 ? off[2] : off[3], r);
                const unsigned m = x == 0 ? ok[0] : x == 1 ? ok[1] : x == 2 ? ok[2] : ok[3];
                raws[i] = (m >> r) & 1 ? ld_stream16(src + o + c * 16) : make_uint4(0, 0, 0, 0);
            };
            locate(0);
#pragma unroll
            for (int i = 0; i < 16; ++i) fetch(i, 0);
            for (int j = 0; j < nblk; ++j) {
                const int st = j % ST;
                char* tile = tiles + st * kTile;
                if (!vacant(j)) break;
                if (side == 0) inform(j % C::SLOTS);
                bool odd = false;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (half == 1 && j + 1 < nblk) locate(j + 1);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int r = half * 64 + 4 * i + (lane >> 3);
                        uint4 lo, hi;
                        codes_to_f16<FMT>(raws[i].x, lo.x, lo.y);
                        codes_to_f16<FMT>(raws[i].y, lo.z, lo.w);
                        codes_to_f16<FMT>(raws[i].z, hi.x, hi.y);
                        codes_to_f16<FMT>(raws[i].w, hi.z, hi.w);
                        if (half == 0) fetch(i, 1);
                        else if (j + 1 < nblk) fetch(i, 0);
                        if (FMT == QF_CACHE_E4M3 && side == 1 && j >= first_draft) {
                            odd |= zero_not_finite<__half>(lo);
                            odd |= zero_not_finite<__half>(hi);
                        }
                        *reinterpret_cast<uint4*>(tile + tile_off(r, 2 * c)) = lo;
                        *reinterpret_cast<uint4*>(tile + tile_off(r, 2 * c + 1)) = hi;
                    }
                }
                if (odd) odd_v = 1;
                proxy_fence();
                mbar_arrive(&full[st]);
            }
        } else {
            const CUtensorMap* map = side ? &tv : &tk;
            const int hi = lane >> 4, c = lane & 15;
            int j = 0;
            for (; j < nblk; ++j) {
                const int st = j % ST, kb = k_begin + j * kRows;
                char* tile = tiles + st * kTile;
                // A block whose keys are all context and all there comes by TMA, a box of
                // `box` slots x 64 dims per lane (K and V alike, 128-byte swizzle)
                bool bulk = box > 0 && j < first_draft && kb + kRows <= k_end;
                int blk = 0, slot0 = 0;
                const int pc = lane >> 1;  // this lane's piece of the block
                if (bulk) {
                    const int key = kb + min(pc * box, kRows - 1);
                    const int lb = a.B.div(key);
                    blk = __ldg(bt + lb);
                    slot0 = key - lb * a.B.d;
                    bulk = __all_sync(kFull, blk >= 0 && blk < a.N);
                }
                if (!bulk) locate(j);
                if (!vacant(j)) break;
                if (bulk) {
                    if (side == 0) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) ok[x] = kFull;
                        inform(j % C::SLOTS);
                    }
                    if (lane == 0) mbar_expect_tx(&full[st], (uint32_t)kTile);
                    else mbar_arrive(&full[st]);
                    __syncwarp();
                    if (pc * box < kRows)
                        tma_page(tile + (lane & 1) * kSlab + pc * box * 128, map, (lane & 1) * 64, slot0, g, blk,
                                 &full[st]);
                    continue;
                }
                if (side == 0) inform(j % C::SLOTS);
                // row by row: chunk c of rows 2 i + hi; the swizzle repeats every four i
                const uint32_t dst = smem_u32(tile) + (uint32_t)((c >> 3) * kSlab + hi * 128);
                const char* from = src + c * 16;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int64_t o = __shfl_sync(kFull, off[x], 2 * i + hi);
                        cp_async16_at(dst + (uint32_t)((x * 32 + 2 * i) * 128 + (((c & 7) ^ ((2 * i & 7) + hi)) << 4)),
                                      from + o, (ok[x] >> (2 * i + hi)) & 1 ? 16 : 0);
                    }
                }
                cp_async_commit();
                cp_async_wait<0>();
                if (side == 1 && j >= first_draft) {  // this lane's own chunks
                    bool odd = false;
                    for (int i = 0; i < 64; ++i) {
                        uint4* at = reinterpret_cast<uint4*>(tile + tile_off(2 * i + hi, c));
                        uint4 v = *at;
                        if (zero_not_finite<MT>(v)) {
                            *at = v;
                            odd = true;
                        }
                    }
                    if (odd) odd_v = 1;
                }
                proxy_fence();
                mbar_arrive(&full[st]);
            }
            // every copy issued has landed before the CTA can leave
            for (int d = max(0, j - ST); d < j; ++d) mbar_wait(&full[d % ST], (d / ST) & 1, nullptr);
        }
    } else if (warp == C::MMA_WARP) {
        // ---- MMA issue: S_t,0 | PV_t,j S_t,j+1 | ...
        if (lane == 0) {
            const uint32_t bf = std::is_same<MT, __nv_bfloat16>::value ? 1u : 0u;
            const uint32_t id_qk = idesc(bf, 0u), id_pv = idesc(bf, 1u);
            const uint32_t qa = smem_u32(base), ka = smem_u32(kbase), va = smem_u32(vbase);
            bool go = mbar_wait(&bars.q_full, 0, abort) && mbar_wait(&bars.k_full[0], 0, abort);
            if (go) {
                tc_fence_after();
                for (int t = 0; t < ntile; ++t) {
                    issue_scores(tmem + t * kRows, qa + t * kTile, ka, id_qk);
                    mma_commit(&bars.s_full[t]);
                }
                mma_commit(&bars.k_empty[0]);
            }
            for (int j = 0; go && j < nblk; ++j) {
                const int st = j % ST, sn = (j + 1) % ST;
                go = mbar_wait(&bars.v_full[st], (j / ST) & 1, abort);
                for (int t = 0; go && t < ntile; ++t) {
                    go = mbar_wait(&bars.p_full[t], j & 1, abort);
                    if (!go) break;
                    tc_fence_after();
                    const uint32_t o = tmem + (uint32_t)((NT + t) * kRows), pt = tmem + (uint32_t)(t * kRows);
                    const uint32_t v = va + (uint32_t)(st * kTile);
#pragma unroll
                    for (int k = 0; k < 8; ++k)  // keys in steps of 16
                        mma_ts(o, pt + 8u * k, sdesc(v + k * 2048, kSlab, 1024), id_pv,
                               (j > 0 || k > 0) ? 1u : 0u);
                    if (j + 1 < nblk) {
                        if (t == 0) {
                            go = mbar_wait(&bars.k_full[sn], ((j + 1) / ST) & 1, abort);
                            if (!go) break;
                            tc_fence_after();
                        }
                        issue_scores(pt, qa + t * kTile, ka + sn * kTile, id_qk);
                        mma_commit(&bars.s_full[t]);
                    }
                }
                mma_commit(&bars.v_empty[st]);
                if (j + 1 < nblk) mma_commit(&bars.k_empty[sn]);
            }
            mma_commit(&bars.o_full);
            mma_commit(&bars.drain);  // every MMA issued has completed before the CTA can leave
            mbar_wait(&bars.drain, 0, nullptr);
        }
    } else if (warp < 4 * ntile) {
        // ---- softmax of tile t, one row per thread
        const int t = warp >> 2, r = tid & (kRows - 1);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t sS = tmem + lanes + (uint32_t)(t * kRows);
        const uint32_t sO = tmem + lanes + (uint32_t)((NT + t) * kRows);
        const T* qrow = reinterpret_cast<const T*>(a.q) + trow_q * a.qt + (int64_t)hq * a.qh;
        const int64_t* mrow = a.mask + trow_q * a.words;
        float rs = sl2;
        {
            using P = Packed<T>;
            float f = 1.f;
            uint32_t flip = 0;
            if (!Q8) {  // rs > 0: a negative scale's sign goes to Q, and 0 becomes as good as 0
                flip = sl2 < 0.f ? 0x80008000u : 0u;
                rs = fabsf(sl2) < 1e-30f ? 1e-30f : fabsf(sl2);
            }
            if constexpr (Q8) {  // a power-of-two factor brings the largest element to [2^14, 2^15)
                uint32_t mx = 0;
                if (live)
                    for (int c = 0; c < 16; ++c) {
                        const uint4 v = ld_shared_ro16(qrow + 8 * c);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            mx = max(mx, max(__float_as_uint(P::lo(word(v, i))) & 0x7fffffffu,
                                             __float_as_uint(P::hi(word(v, i))) & 0x7fffffffu));
                    }
                const int e = min(max((int)(mx >> 23) - 127, -100), 127);
                f = __int_as_float((127 + 14 - e) << 23);
                rs = sl2 * __int_as_float((127 - 14 + e) << 23);
            }
            for (int c = 0; c < 16; ++c) {
                uint4 v = live ? ld_shared_ro16(qrow + 8 * c) : make_uint4(0, 0, 0, 0);
                if constexpr (Q8) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        set_word(v, i, MP::pack(P::lo(word(v, i)) * f, P::hi(word(v, i)) * f));
                }
                if (!Q8) v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
                *reinterpret_cast<uint4*>(base + t * kTile + tile_off(r, c)) = v;
            }
            proxy_fence();
            mbar_arrive(&bars.q_full);
        }
        float m = -INFINITY, l = 0.f;  // reference maximum and the sum against it
        float lvtop = -INFINITY;       // largest log2 v-scale so far
        bool got = true;
        for (int j = 0; j < nblk; ++j) {
            const int slot = j % C::SLOTS, kb = k_begin + j * kRows;
            got = mbar_wait(&bars.info_full[slot], (j / C::SLOTS) & 1, abort) &&
                  mbar_wait(&bars.s_full[t], j & 1, abort);
            if (!__all_sync(kFull, got)) {
                got = false;
                break;
            }
            tc_fence_after();
            uint32_t see[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                see[q] = live ? valid[slot][q] : 0u;
                if (j >= first_draft && live) see[q] &= tree_bits32(mrow, a.words, kb + 32 * q - w.ctx);
            }
            const bool masked = __any_sync(kFull, (see[0] & see[1] & see[2] & see[3]) != kFull);
            // Scores in log2 units, with V's scale where there is one: 16-bit rows x * rs,
            // rs > 0 (a negative scale is in Q), so the maximum is that of x.
            auto score = [&](float x, int c) -> float {
                if constexpr (Q8) return fmaf(x * rs, sk[slot][c], sl[slot][c]);
                else return x;
            };
            bool wide = false;
            if constexpr (Q8) {
                lvtop = fmaxf(lvtop, srange[slot][1]);
                wide = lvtop - srange[slot][0] > kScaleRange;
            }
            // One pass over S against the reference m, P in registers, the block's maximum on
            // the side.  While no row's maximum has grown past 2^8 (but for the first blocks,
            // nearly always) P stands; else the reference moves, O and l with it, and
            // the pass is made again over S, which P has not touched yet.
            uint32_t pk[64];
            float sum;
            for (int turn = 0;; ++turn) {
                const float mref = m == -INFINITY ? 0.f : m;
                float mx0 = -INFINITY, mx1 = -INFINITY;
                float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
                constexpr int NX = NT == 2 ? 2 : 1;  // registers allow: the next quarter's load in flight
                uint32_t x[NX][32];
                tmem_ld32(sS, x[0]);
                tmem_wait_ld();
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (NX == 2 && q < 3) tmem_ld32(sS + 32 * (q + 1), x[(q + 1) % NX]);
                    uint32_t* xs = x[q % NX];
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!((see[q] >> e) & 1)) xs[e] = __float_as_uint(-INFINITY);
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const int c = 32 * q + e;
                        const float x0 = __uint_as_float(xs[e]), x1 = __uint_as_float(xs[e + 1]);
                        float t0, t1;
                        if constexpr (Q8) {
                            t0 = score(x0, c);
                            t1 = score(x1, c + 1);
                            if (masked) {  // an unseen key's scales may be anything
                                if (x0 == -INFINITY) t0 = -INFINITY;
                                if (x1 == -INFINITY) t1 = -INFINITY;
                            }
                            mx0 = max3(mx0, t0, t1);
                            t0 -= mref;
                            t1 -= mref;
                        } else {
                            if (e & 2) mx1 = max3(mx1, x0, x1);
                            else mx0 = max3(mx0, x0, x1);
                            fma2(t0, t1, x0, x1, rs, -mref);
                        }
                        const float p0 = ex2(t0), p1 = ex2(t1);
                        if constexpr (Q8) {
                            if (!wide) {
                                s0 = fmaf(p0, !masked || t0 != -INFINITY ? sr_[slot][c] : 0.f, s0);
                                s1 = fmaf(p1, !masked || t1 != -INFINITY ? sr_[slot][c + 1] : 0.f, s1);
                            } else {
                                s0 += t0 == -INFINITY ? 0.f : ex2(t0 - sl[slot][c]);
                                s1 += t1 == -INFINITY ? 0.f : ex2(t1 - sl[slot][c + 1]);
                            }
                        } else if (e & 2) {
                            add2(s2, s3, p0, p1);
                        } else {
                            add2(s0, s1, p0, p1);
                        }
                        pk[16 * q + (e >> 1)] = MP::pack(p0, p1);
                    }
                    if (NX == 1 && q < 3) tmem_ld32(sS + 32 * (q + 1), x[0]);
                    if (q < 3) tmem_wait_ld();
                }
                sum = (s0 + s1) + (s2 + s3);
                const float mx = fmaxf(mx0, mx1) * (Q8 ? 1.f : rs);
                const bool move = turn == 0 && (mx > m + kKeepLog2 || (m == -INFINITY && mx > -INFINITY));
                if (!__any_sync(kFull, move)) break;
                // the block before's P V is done: S of this block was issued after it
                const float corr = move ? ex2(m - mx) : 1.f;
                if (j > 0) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t o[32];
                        tmem_ld32(sO + 32 * q, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                        tmem_st32(sO + 32 * q, o);
                    }
                }
                l *= corr;
                if (move) m = mx;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) tmem_st16(sS + 16 * q, pk + 16 * q);
            l += sum;
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bars.p_full[t]);
        }
        got = got && mbar_wait(&bars.o_full, 0, abort);
        if (__all_sync(kFull, got)) {
            tc_fence_after();
            const bool whole = w.nparts == 1;
            const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
            float* part = a.ws + ((trow_q * a.Hq + hq) * a.P + p) * (kD + 2);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t o[32];
                tmem_ld32(sO + 32 * q, o);
                tmem_wait_ld();
                if (live && whole) {
                    using P = Packed<T>;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint4 v;
                        v.x = P::pack(__uint_as_float(o[8 * c]) * inv, __uint_as_float(o[8 * c + 1]) * inv);
                        v.y = P::pack(__uint_as_float(o[8 * c + 2]) * inv, __uint_as_float(o[8 * c + 3]) * inv);
                        v.z = P::pack(__uint_as_float(o[8 * c + 4]) * inv, __uint_as_float(o[8 * c + 5]) * inv);
                        v.w = P::pack(__uint_as_float(o[8 * c + 6]) * inv, __uint_as_float(o[8 * c + 7]) * inv);
                        st16(orow + 32 * q + 8 * c, v);
                    }
                } else if (live) {
#pragma unroll
                    for (int e = 0; e < 32; e += 2)
                        *reinterpret_cast<float2*>(part + 32 * q + e) =
                            make_float2(__uint_as_float(o[e]), __uint_as_float(o[e + 1]));
                }
                __syncwarp();  // the next quarter's load is warp-wide
            }
            if (live && !whole) *reinterpret_cast<float2*>(part + kD) = make_float2(m, l);
            if (live && *static_cast<volatile int*>(&odd_v)) {  // (set before the last v_full, which o_full follows)
                const int j0 = k_begin + min(first_draft, nblk) * kRows;
                if (whole) add_not_finite<T, FMT, T>(a, bt, g, w.ctx, mrow, qrow, sl2, m, j0, k_end, orow);
                else add_not_finite<T, FMT, float>(a, bt, g, w.ctx, mrow, qrow, sl2, m, j0, k_end, part);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (tid == 0 && abort_flag) flag(a.status, QF_FLAG_TIMEOUT);
    if (warp == C::MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS)
                     : "memory");
    }
}

// A map over a 16-bit cache (128 dims, B slots, Hkv heads, N blocks), boxes of 64 dims x `box` slots.
bool page_map(CUtensorMap* map, const char* ptr, const TreeDev& a, int bf16, int box) {
    PFN_cuTensorMapEncodeTiled fn = tensor_map_encode();
    if (!fn || a.N <= 0) return false;
    const cuuint64_t dims[4] = {kD, (cuuint64_t)a.B.d, (cuuint64_t)a.Hkv, (cuuint64_t)a.N};
    const cuuint64_t strides[3] = {(cuuint64_t)a.c2 * 2, (cuuint64_t)a.c1 * 2, (cuuint64_t)a.c0 * 2};
    const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1};
    const cuuint32_t step[4] = {1, 1, 1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
              const_cast<char*>(ptr), dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int FMT, int NT>
int launch_nt(const TreeDev& a, cudaStream_t stream) {
    constexpr auto kernel = tree_tc_kernel<T, FMT, NT>;
    const int rc = allow_smem<kernel>(TreeTc<NT>::SMEM);
    if (rc) return rc;
    const int64_t groups = ceil_div((int64_t)a.max_tree * a.G, NT * kRows);
    if (groups * a.Hkv > 65535) return QF_ERR_UNSUPPORTED;
    // The largest power of two that divides a page and a block: a piece never crosses a
    // page.  Below 8 (or where the cache's shape has no map) rows come one by one.
    CUtensorMap tk{}, tv{};
    int box = 0;
    if (FMT == QF_CACHE_PLAIN) {
        const int bf16 = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
        box = std::min(a.B.d & -a.B.d, kRows);
        if (box < 8 || !page_map(&tk, a.kc, a, bf16, box) || !page_map(&tv, a.vc, a, bf16, box)) box = 0;
    }
    kernel<<<dim3((unsigned)a.P, (unsigned)(groups * a.Hkv), (unsigned)a.S), TreeTc<NT>::THREADS,
             TreeTc<NT>::SMEM, stream>>>(a, tk, tv, box);
    return check_launch();
}

template <typename T, int FMT>
int launch_fmt(const TreeDev& a, int tiles, cudaStream_t stream) {
    return tiles == 1 ? launch_nt<T, FMT, 1>(a, stream) : launch_nt<T, FMT, 2>(a, stream);
}

template <typename T>
int launch_t(const TreeDev& a, int format, int tiles, cudaStream_t stream) {
    switch (format) {
    case QF_CACHE_PLAIN: return launch_fmt<T, QF_CACHE_PLAIN>(a, tiles, stream);
    case QF_CACHE_E4M3: return launch_fmt<T, QF_CACHE_E4M3>(a, tiles, stream);
    default: return launch_fmt<T, QF_CACHE_INT8>(a, tiles, stream);
    }
}

}  // namespace

int launch_tree_tc(const TreeDev& a, int dtype, int format, int tiles, cudaStream_t stream) {
    return dtype == QF_F16 ? launch_t<__half>(a, format, tiles, stream)
                           : launch_t<__nv_bfloat16>(a, format, tiles, stream);
}

}  // namespace qf
