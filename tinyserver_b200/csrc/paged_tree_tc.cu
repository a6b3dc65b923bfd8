// Paged attention for many query rows per kv head (a tree's tokens x G), 16-bit
// queries, head_dim 128, on the 5th-generation tensor cores.
//
// A CTA takes NT tiles of 128 rows of one (sequence, kv head) and a stretch of
// the keys in blocks of 128.  Both products run on tcgen05.mma with S, P and O in
// tensor memory, P over the S it came from:
//   S_t = Q K_j^T     Q, K in shared memory (128-byte swizzle)
//   softmax of row r by thread r of warpgroup t, whose tensor-memory lane the row
//   is; P_t back over the first half of S_t
//   O_t += P_t V_j    A = P_t from tensor memory, V in shared memory
// There are two S, two O and two softmax warpgroups.  NT = 2 (more than 128 rows):
// warpgroup t has tile t; K and V meet 256 rows, and tile 0's softmax overlaps tile
// 1's products.  NT = 1: the warpgroups take turns at the one tile's blocks, each
// with a maximum, a sum and an O of its own, which the end of the item joins; so one
// block's products and copies overlap the softmax of the block before.
// P goes back by halves of a block: the first half's products run during the
// second's softmax.  (Scores by halves too, taking turns in S_t, overlap better on
// paper, but 64 columns cost the tensor core as much as 128: 511 cycles for a tile's
// eight steps against 515.)
// Roles: 8 softmax warps, one MMA thread, and loaders: one warp each for K and V, or
// two (NT = 1), every other block one's.  16-bit pages come by TMA, one box per
// lane, where a block's keys are all context; else (the drafted keys, the tail, pages
// whose size is no multiple of 8) row by row with cp.async.  8-bit rows land in half
// of their tile and are converted to fp16 (exact) in place.
//
// What bounds it: a block is 64 KB of 16-bit K and V, ~2800 cycles of an SM's
// share of HBM; a tile's softmax is 16384 exponentials, 1024 cycles of the MUFU,
// and its products 1024 cycles of the tensor core.
//  * Up to 128 rows, 16-bit rows: by HBM's latency, with 128 KB of K and V stages per
//    SM: 32 trees of 16 nodes x 4 heads at 4096 context keys, 8 kv heads: 109 us, 5.0
//    TB/s (two CTAs per SM with one stage each and halves of a block in turn: 127 us).
//  * 8-bit rows: by the softmax warps' dependent instructions (two warps per scheduler;
//    36% of the issue slots used): a half block takes 2300 cycles, against 1100 over
//    16-bit rows, for the scales' loads and products.  The same trees over e4m3: 158 us
//    (182 us then); 32 trees of 32 nodes at up to 8191 context keys: 208 to 238 us, from
//    process to process.
//  * More than 128 rows: by the chain of products and softmax, ~4100 cycles a block of
//    two tiles; 64 trees of 64 nodes x 4 heads at up to 8191 context keys: 332 to 345
//    us, 880 to 920 TFLOP/s (as single tiles, which read K and V twice, 445 us against 350
//    then).
// Registers moved from the loaders to the softmax (88 and 168 a thread instead of 128)
// cost more in the loaders than they gained: 154 -> 206 us.
//
// Quantised rows: the codes go into the products as they are.  K's scale multiplies
// the score, V's (times 2^x, x of the segment's first block) the probability before
// its one rounding; the sum takes the probability alone.  A block with a scale
// that 2^x does not bring into [2^-6, 2^3] has V's scale in the exponent instead,
// p' = 2^(t + log2 vs + x - m), m being the maximum of that (see kLeastLog2), so that p' fits fp16
// whatever the scales' range.
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
// What beginning and ending an item costs, in blocks.  64 trees of 64, 16 of 16 over
// 16-bit rows, 32 of 32 over e4m3: 347, 48.7, 214 us; with 2: 370, 53.5, 234; 8: 357, 51.9, 213.
constexpr int kItemBlocks = 4;
// The probabilities' range.  When a row's reference moves, its largest p becomes 2^ROOM; it
// moves again once p would pass 2^TOP, 2^8 more (2^6 more, over codes: 212 -> 239 us).  fp16
// ends at 2^-24 and 2^16, so over fp16 rows TOP is 15, and over codes 12, since V's scales
// (times 2^x), 2^-6 to 2^3 of them, go into P before its rounding.  So p keeps fp16's
// precision down to 2^-21 of a row's largest, over codes 2^-18, and something down to 2^-31
// and 2^-28.  (With ROOM 0, 2^18 keys at 2^-25.5, all of a row's output beside a key whose V
// is 0, gave 0.)
template <bool Q8, typename MT>
struct PRange {
    static constexpr bool H = std::is_same<MT, __half>::value;
    static constexpr float TOP = Q8 ? 12.f : H ? 15.f : 8.f;
    static constexpr float ROOM = Q8 ? 4.f : H ? 7.f : 0.f;
};
constexpr float kScaleLow = -6.f, kScaleTop = 3.f;  // log2 of those scales
// In the reference a V scale (times 2^x) counts as 2^-85 at least (a row never written has 0):
// the sum, which has no scale in it, grows by 2^(85 + TOP) a key at most.
constexpr float kLeastLog2 = -85.f;

template <int NT>
struct TreeTc {
    static constexpr int ST = 2;              // K and V stages
    static constexpr int LW = NT == 1 ? 2 : 1;  // loader warps of K, and of V: block n is warp n % LW's
    static constexpr int SOFT = 256;          // softmax threads
    static constexpr int MMA_WARP = 8, LOAD_WARP = 9;  // K's, then V's
    static constexpr int THREADS = SOFT + 32 + 64 * LW;
    static constexpr int SLOTS = 2 * ST;      // blocks whose scales and valid bits are kept
    static constexpr int SMEM = (NT + 2 * ST) * kTile + 1024;
};
constexpr uint32_t kCols = 512;  // tensor memory: S_t at 128 t, O_t at 256 + 128 t

struct TreeBars {
    uint64_t q_full;
    uint64_t k_full[2], v_full[2], k_empty[2], v_empty[2];
    uint64_t info_full[4];  // a block's valid bits and scales
    uint64_t s_full[2], p_full[2][2];  // P by halves of a block
    uint64_t pv_done[2], o_full, drain;
    uint64_t raw[4];  // a tile that its loader still works on has landed
};

// By the softmax warps, all together: whether `ok` holds in every thread.
__device__ __forceinline__ bool soft_all(bool ok) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"((uint32_t)ok)
        : "memory");
    return all != 0;
}

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

// Whether two 16-bit values hold an infinity or a NaN: an exponent of all ones
// carries into the sign's place when one is added to it.
template <typename T>
__device__ __forceinline__ uint32_t odd_pair(uint32_t w) {
    constexpr bool H = std::is_same<T, __half>::value;
    return ((w & (H ? 0x7c007c00u : 0x7f807f80u)) + (H ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}

// Infinities and NaN of 8 16-bit values set to zero.
template <typename T>
__device__ __forceinline__ void zero_not_finite(uint4& v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w = word(v, i);
        const uint32_t o = odd_pair<T>(w);
        if (o & 0x8000u) w &= 0xffff0000u;
        if (o & 0x80000000u) w &= 0xffffu;
        set_word(v, i, w);
    }
}

// By one warp: rows [r0, r1) of a V tile looked through, and infinities and NaN in
// them set to zero; whether there were any.
template <typename T>
__device__ __forceinline__ bool clean_rows(char* tile, int r0, int r1, int lane) {
    const int c = lane & 15, hi = lane >> 4;
    uint32_t odd = 0;
    for (int r = r0; r < r1; r += 16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int rr = min(r + 2 * i + hi, r1 - 1);
            const uint4 v = *reinterpret_cast<const uint4*>(tile + tile_off(rr, c));
            odd |= odd_pair<T>(v.x) | odd_pair<T>(v.y) | odd_pair<T>(v.z) | odd_pair<T>(v.w);
        }
    }
    if (!__any_sync(kFull, odd != 0)) return false;
    for (int r = r0 + hi; r < r1; r += 2) {
        uint4* at = reinterpret_cast<uint4*>(tile + tile_off(r, c));
        uint4 v = *at;
        zero_not_finite<T>(v);
        *at = v;
    }
    return true;
}

// By one warp: a tile's codes, which landed in its second slab (a row's 128 codes are
// as long as half a row of fp16), into the fp16 tile, in place: a row is read by
// eight lanes before any of them writes.  (The lanes of a row's second half take the
// row beside it, whose swizzle puts their chunks in other banks.)  EDGE: rows from nk
// on are zero, and infinities and NaN in rows from d0 on are set to zero; whether
// there were any.
template <int FMT, bool EDGE>
__device__ __forceinline__ bool expand(char* tile, int nk, int d0, int lane) {
    const int c = lane & 7, r4 = (lane >> 3) ^ (c >> 2);
    uint32_t odd = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < 32; i0 += 8) {
        uint4 raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            raw[i] = *reinterpret_cast<const uint4*>(tile + kSlab + (4 * (i0 + i) + r4) * 128 + c * 16);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = 4 * (i0 + i) + r4;
            uint4 lo, hi;
            codes_to_f16<FMT>(raw[i].x, lo.x, lo.y);
            codes_to_f16<FMT>(raw[i].y, lo.z, lo.w);
            codes_to_f16<FMT>(raw[i].z, hi.x, hi.y);
            codes_to_f16<FMT>(raw[i].w, hi.z, hi.w);
            if constexpr (EDGE) {
                if (r >= nk) lo = hi = make_uint4(0, 0, 0, 0);
                if (FMT == QF_CACHE_E4M3 && r >= d0) {
                    odd |= odd_pair<__half>(lo.x) | odd_pair<__half>(lo.y) | odd_pair<__half>(lo.z) |
                           odd_pair<__half>(lo.w) | odd_pair<__half>(hi.x) | odd_pair<__half>(hi.y) |
                           odd_pair<__half>(hi.z) | odd_pair<__half>(hi.w);
                    zero_not_finite<__half>(lo);
                    zero_not_finite<__half>(hi);
                }
            }
            *reinterpret_cast<uint4*>(tile + tile_off(r, 2 * c)) = lo;
            *reinterpret_cast<uint4*>(tile + tile_off(r, 2 * c + 1)) = hi;
        }
        __syncwarp();
    }
    return EDGE && __any_sync(kFull, odd != 0);
}

// q . k over the 128 dims on the CUDA cores, k a cache row.
template <typename T, int FMT>
__device__ float dot_row(const T* q, const char* k) {
    float acc = 0.f;
#pragma unroll 4
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
// finite part was).  Keys [j0, k_end), one row per thread, its columns [d0, d1).
template <typename T, int FMT, typename O>
__device__ __noinline__ void add_not_finite(const TreeDev& a, const int32_t* bt, int g, int ctx,
                                            const int64_t* mrow, const T* q, float sl2, float mref,
                                            int j0, int k_end, int d0, int d1, O* out) {
    for (int j = j0; j < k_end; ++j) {
        if (!((tree_bits32(mrow, a.words, j - ctx)) & 1u)) continue;
        int64_t row, srow;
        if (!key_place(a, bt, g, j, row, srow)) continue;
        float p = -1.f;
#pragma unroll 1
        for (int d = d0; d < d1; ++d) {
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

// 8 consecutive columns of this thread's lane.
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// One lane of a converged warp, known as such to the assembler: the products'
// operands, alike in all lanes, then stay in uniform registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is != 0;
}

// Shared-memory descriptors as their two words: the low one is the address in 16
// bytes and the leading offset, so stepping through a tile is one add, and the
// issuing thread, which shares its scheduler with softmax warps, has few
// instructions per product.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) {
    return (uint32_t)sdesc(addr, lbo, 1024);
}
__device__ __forceinline__ uint64_t desc_of(uint32_t lo) {
    constexpr uint64_t hi = (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;  // as sdesc(., ., 1024)
    return hi | lo;
}

// S = Q K^T, from the descriptors of Q's and K's first step: head_dim in steps of 16,
// 32 bytes on in a slab, then the second slab.
__device__ __forceinline__ void issue_scores(uint32_t d, uint32_t q, uint32_t k, uint32_t id) {
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
        const uint32_t off = (uint32_t)((kk >> 2) * (kSlab >> 4) + (kk & 3) * 2);
        mma_ss(d, desc_of(q + off), desc_of(k + off), id, kk > 0 ? 1u : 0u);
    }
}

template <typename T, int FMT, int NT>
__global__ void __launch_bounds__(TreeTc<NT>::THREADS, 1)
    tree_tc_kernel(const TreeDev a, const __grid_constant__ CUtensorMap tk,
                   const __grid_constant__ CUtensorMap tv, int box) {
    using C = TreeTc<NT>;
    constexpr bool Q8 = FMT != QF_CACHE_PLAIN;
    using MT = typename std::conditional<Q8, __half, T>::type;
    using MP = Packed<MT>;
    using PR = PRange<Q8, MT>;
    constexpr int ST = C::ST, LW = C::LW;
    constexpr bool TURNS = NT == 1;  // the warpgroups take turns at one tile's blocks
    constexpr int STEP = TURNS ? 2 : 1;  // between a warpgroup's blocks

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    extern __shared__ __align__(1024) char dsm[];
    __shared__ TreeBars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, odd_v;  // odd_v: the last segment whose drafted V was not finite, from 1
    __shared__ int scratch[34];
    __shared__ __align__(16) uint32_t valid[C::SLOTS][4];
    // of a block's keys: k-scale, v-scale * 2^x, log2 of that; whether the block's all are
    // near 1; x
    __shared__ __align__(16) float sk[Q8 ? C::SLOTS : 1][Q8 ? kRows : 4], sv[Q8 ? C::SLOTS : 1][Q8 ? kRows : 4],
        sl[Q8 ? C::SLOTS : 1][Q8 ? kRows : 4];
    __shared__ int snear[C::SLOTS], sexp[C::SLOTS];
    __shared__ float stat[TURNS ? 3 : 1][TURNS ? 256 : 1];  // m, l, 2^-x of the softmax threads
    __shared__ uint32_t qtop[TURNS && Q8 ? 256 : 1];        // largest magnitude in a row of Q's slab
    volatile int* abort = &abort_flag;

    const uint32_t raw = smem_u32(dsm);
    char* base = dsm + (((raw + 1023u) & ~1023u) - raw);
    char* const kbase = base + NT * kTile;
    char* const vbase = kbase + ST * kTile;
    if (tid == 0) {
        mbar_init(&bars.q_full, C::SOFT);
        for (int i = 0; i < ST; ++i) {
            mbar_init(&bars.k_full[i], 32);
            mbar_init(&bars.v_full[i], 32);
            mbar_init(&bars.k_empty[i], 1);
            mbar_init(&bars.v_empty[i], 1);
        }
        for (int i = 0; i < C::SLOTS; ++i) mbar_init(&bars.info_full[i], 32);
        for (int t = 0; t < 2; ++t) {
            mbar_init(&bars.s_full[t], 1);
            for (int h = 0; h < 2; ++h) mbar_init(&bars.p_full[t][h], kRows);
            mbar_init(&bars.pv_done[t], 1);
        }
        mbar_init(&bars.o_full, 1);
        mbar_init(&bars.drain, 1);
        for (int i = 0; i < 2 * LW; ++i) mbar_init(&bars.raw[i], 1);
        abort_flag = 0;
        odd_v = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == C::MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_slot)),
                     "r"(kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const float sl2 = a.scale * 1.4426950408889634f;

    // launched with programmatic dependent launch: what is above overlaps the kernel before
    pdl_wait();
    pdl_trigger();
    // every role walks the same segments; barrier phases run on across them
    TreeWalk<kRows, NT * kRows, kItemBlocks> walk;
    walk.begin(a, scratch);
    zero_unowned_rows<T, kD>(a);
    if (tid == 0) walk.record(a);
    TreeSeg sg{};
    auto blocks_of = [&]() { return (sg.k_end - sg.k_begin + kRows - 1) / kRows; };
    auto tiles_of = [&]() {
        return min(NT, (sg.w.n * a.G - sg.rg * NT * kRows + kRows - 1) / kRows);
    };
    // the first block that a row may not see whole
    auto draft_of = [&](int nblk) { return a.cu ? max(0, (sg.w.ctx - sg.k_begin) / kRows) : nblk; };

    if (warp >= C::LOAD_WARP) {
        // ---- loaders: K's warps, then V's; every LW-th block of all segments is one's
        const int side = (warp - C::LOAD_WARP) / LW, turn = (warp - C::LOAD_WARP) % LW;
        const char* src = side ? a.vc : a.kc;
        char* const tiles = side ? vbase : kbase;
        uint64_t* full = side ? bars.v_full : bars.k_full;
        uint64_t* empty = side ? bars.v_empty : bars.k_empty;
        const int32_t* bt = nullptr;
        // lane l: keys l, l + 32, l + 64, l + 96 of a block
        int64_t off[4];
        unsigned ok[4];
        float ks[4], vs[4];
        auto locate = [&](int j) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int key = sg.k_begin + j * kRows + x * 32 + lane;
                int64_t srow = 0;
                off[x] = 0;
                ks[x] = 0.f;
                vs[x] = 1.f;
                const bool in = key < sg.k_end && key_place(a, bt, sg.g, key, off[x], srow);
                ok[x] = __ballot_sync(kFull, in);
                if (!Q8) off[x] *= 2;  // bytes
                if (Q8 && side == 0 && in) {
                    ks[x] = __ldg(a.ks + srow);
                    vs[x] = __ldg(a.vs + srow);
                }
            }
        };
        // The same scales for a block whose pages are all there, in two steps with the work
        // on another block between them: the keys' pages, then the scales.
        int page[4];
        auto look_scales = [&](int j) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int key = sg.k_begin + j * kRows + x * 32 + lane;
                page[x] = key < sg.k_end ? __ldg(bt + a.B.div(key)) : -1;
            }
        };
        auto load_scales = [&](int j) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int key = sg.k_begin + j * kRows + x * 32 + lane;
                ks[x] = 0.f;
                vs[x] = 1.f;
                if (page[x] >= 0 && page[x] < a.N) {
                    const int64_t srow = (int64_t)page[x] * a.s0 + (int64_t)sg.g * a.s1 +
                                         (int64_t)(key - a.B.div(key) * a.B.d) * a.s2;
                    ks[x] = __ldg(a.ks + srow);
                    vs[x] = __ldg(a.vs + srow);
                }
            }
        };
        // What the softmax needs to know of a block's keys.  The slot's last reader, the
        // softmax SLOTS blocks ago, is done: S of ST blocks ago (whose K was in this
        // stage) came after it.
        int vexp = 0;  // x
        auto inform = [&](int slot, bool first) {
            if (lane == 0) *reinterpret_cast<uint4*>(valid[slot]) = make_uint4(ok[0], ok[1], ok[2], ok[3]);
            if constexpr (Q8) {
                if (first) {
                    float top = 0.f;
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        if ((ok[x] >> lane) & 1) top = fmaxf(top, vs[x]);
                    top = warp_max(top);
                    vexp = 127 - min(max((int)(__float_as_uint(top) >> 23), 127 - 100), 127 + 100);
                }
                const float f = __int_as_float((127 + vexp) << 23);
                bool near = true;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float v = vs[x] * f, lv = log2f(vs[x]) + (float)vexp;
                    if ((ok[x] >> lane) & 1) near = near && lv >= kScaleLow && lv <= kScaleTop;  // (a NaN is not near)
                    sk[slot][x * 32 + lane] = ks[x];
                    sv[slot][x * 32 + lane] = v;
                    sl[slot][x * 32 + lane] = lv;
                }
                near = __all_sync(kFull, near);
                if (lane == 0) snear[slot] = near, sexp[slot] = vexp;
            }
            __syncwarp();
            mbar_arrive(&bars.info_full[slot]);
        };
        // the stage of block n (of all segments) may be refilled; the whole warp learns the same
        auto vacant = [&](int n) -> bool {
            return __all_sync(kFull, n < ST || mbar_wait(&empty[n % ST], ((n / ST) - 1) & 1, abort));
        };
        bool go = true;
        int seq_no = 0;  // segments begun
        const CUtensorMap* map = side ? &tv : &tk;
        const int hi = lane >> 4, c = lane & 15;
        // this lane's piece of a block: `box` slots of one page, 64 dims of them or all codes
        const int pc = Q8 ? lane : lane >> 1;
        int n0 = 0, last = -1;  // the segment's first block of all segments', and the last one begun here
        int raw = 0;            // tiles worked on
        uint64_t* const landed = &bars.raw[warp - C::LOAD_WARP];
        int blk = 0, slot0 = 0;
        auto look = [&](int j) {  // the page and first slot of this lane's piece of block j
            const int kb = sg.k_begin + j * kRows;
            const int key = kb + (pc * box < min(kRows, sg.k_end - kb) ? pc * box : 0);
            const int lb = a.B.div(key);
            blk = __ldg(bt + lb);
            slot0 = key - lb * a.B.d;
        };
        while (go && walk.next(a, sg)) {
            ++seq_no;
            bt = a.bt + (int64_t)sg.s * a.bts;
            const int nblk = blocks_of(), k_end = sg.k_end;
            const int j0 = LW == 1 ? 0 : (turn + n0) & 1;
            if (box > 0 && j0 < nblk) {
                look(j0);
                if (Q8 && side == 0) {
                    look_scales(j0);
                    load_scales(j0);
                }
            }
            for (int j = j0; j < nblk; j += LW) {
                const int n = n0 + j, st = n % ST, kb = sg.k_begin + j * kRows, nk = min(kRows, k_end - kb);
                char* tile = tiles + st * kTile;
                // rows of V that some query row may not see
                const int d0 = a.cu ? max(0, sg.w.ctx - kb) : kRows;
                bool bulk = box > 0;
                const bool mine = pc * box < nk;
                if (bulk) bulk = __all_sync(kFull, blk >= 0 && blk < a.N);
                if (!bulk) locate(j);
                if (!vacant(n)) {
                    go = false;
                    break;
                }
                last = n;
                // whether this warp works on the tile before the tensor core may have it
                const bool work = Q8 || (side == 1 && (nk < kRows || d0 < nk));
                if (bulk) {
                    // (K behind the last key may hold anything: those columns are masked)
                    uint64_t* bar = work ? landed : &full[st];
                    const uint32_t bytes = (uint32_t)((nk + box - 1) / box * box) * (Q8 ? 128u : 256u);
                    if (lane == 0) mbar_expect_tx(bar, bytes);
                    else if (!work) mbar_arrive(bar);
                    __syncwarp();
                    if (mine) {
                        if constexpr (Q8)
                            tma_page(tile + kSlab + pc * box * 128, map, 0, slot0, sg.g, blk, bar);
                        else
                            tma_page(tile + (lane & 1) * kSlab + pc * box * 128, map, (lane & 1) * 64, slot0, sg.g, blk,
                                     bar);
                    }
                    if (j + LW < nblk) look(j + LW);
                    if (side == 0) {  // meanwhile, what the softmax needs to know
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            ok[x] = nk >= 32 * (x + 1) ? kFull : nk > 32 * x ? (1u << (nk - 32 * x)) - 1u : 0u;
                        inform(n % C::SLOTS, j == j0);
                        if (Q8 && j + LW < nblk) look_scales(j + LW);
                    }
                    if (!work) continue;
                    if (!__all_sync(kFull, mbar_wait(bar, raw++ & 1, nullptr))) {
                        go = false;
                        break;
                    }
                    if (!Q8)
                        for (int r = nk + hi; r < kRows; r += 2)
                            *reinterpret_cast<uint4*>(tile + tile_off(r, c)) = make_uint4(0, 0, 0, 0);
                } else if constexpr (Q8) {  // row by row, 16 codes a lane
                    if (box > 0 && j + LW < nblk) {
                        look(j + LW);
                        if (side == 0) look_scales(j + LW);
                    }
                    const uint32_t dst = smem_u32(tile) + (uint32_t)(kSlab + (lane >> 3) * 128 + (lane & 7) * 16);
#pragma unroll
                    for (int x = 0; x < 4; ++x)
#pragma unroll 1
                        for (int i = 0; i < 8; ++i) {
                            const int r = 4 * i + (lane >> 3);
                            const int64_t o = __shfl_sync(kFull, off[x], r);
                            cp_async16_at(dst + (uint32_t)((x * 32 + 4 * i) * 128), src + o + (lane & 7) * 16,
                                          (ok[x] >> r) & 1 ? 16 : 0);
                        }
                    cp_async_commit();
                    if (side == 0) inform(n % C::SLOTS, j == j0);
                    cp_async_wait<0>();
                    __syncwarp();
                } else {  // chunk c of rows 2 i + hi; the swizzle repeats every four i
                    if (box > 0 && j + LW < nblk) look(j + LW);
                    const uint32_t dst = smem_u32(tile) + (uint32_t)((c >> 3) * kSlab + hi * 128);
                    const char* from = src + c * 16;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
#pragma unroll 4
                        for (int i = 0; i < 16; ++i) {
                            const int64_t o = __shfl_sync(kFull, off[x], 2 * i + hi);
                            cp_async16_at(dst + (uint32_t)((x * 32 + 2 * i) * 128 + (((c & 7) ^ ((2 * i & 7) + hi)) << 4)),
                                          from + o, (ok[x] >> (2 * i + hi)) & 1 ? 16 : 0);
                        }
                    }
                    cp_async_commit();
                    if (side == 0) inform(n % C::SLOTS, j == j0);
                    cp_async_wait<0>();
                    __syncwarp();
                }
                if constexpr (Q8) {
                    if (side == 0 || (nk == kRows && d0 >= kRows)) expand<FMT, false>(tile, nk, d0, lane);
                    else if (expand<FMT, true>(tile, nk, d0, lane)) atomicMax(&odd_v, seq_no);
                } else {
                    if (work && d0 < nk && clean_rows<MT>(tile, d0, nk, lane)) atomicMax(&odd_v, seq_no);
                }
                proxy_fence();
                mbar_arrive(&full[st]);
                if (Q8 && side == 0 && box > 0 && j + LW < nblk) load_scales(j + LW);
            }
            n0 += nblk;
        }
        // every copy issued has landed before the CTA can leave
        for (int d = last - (ST - LW); d <= last; d += LW)
            if (d >= 0) mbar_wait(&full[d % ST], (d / ST) & 1, nullptr);
    } else if (warp == C::MMA_WARP) {
        // ---- MMA issue, the warp together and one lane for it: S_t,0 | PV_t,j by the two
        // halves of P, S_t,j+1 | ...
        const uint32_t bf = std::is_same<MT, __nv_bfloat16>::value ? 1u : 0u;
        const uint32_t id_qk = idesc(bf, 0u), id_pv = idesc(bf, 1u);
        const uint32_t qa = desc_lo(smem_u32(base), 16), ka = desc_lo(smem_u32(kbase), 16);
        const uint32_t va = desc_lo(smem_u32(vbase), kSlab);
        bool go = true;
        auto wait = [&](uint64_t* bar, uint32_t phase) {
            go = __all_sync(kFull, go && mbar_wait(bar, phase & 1, abort));
            tc_fence_after();
        };
        uint32_t n = 0, seg = 0;  // blocks, segments with keys so far
        uint32_t uses[2] = {};    // blocks of each tile so far (turns: n / 2)
        while (go && walk.next(a, sg)) {
            const int nblk = blocks_of(), ntile = TURNS ? 1 : tiles_of();
            if (nblk == 0) continue;
            wait(&bars.q_full, seg);
            // scores of block bn into S_t; K's stage is free once the last tile's have been issued
            auto scores = [&](uint32_t bn, int t) {
                if (TURNS || t == 0) wait(&bars.k_full[bn % ST], bn / ST);
                if (!go) return;
                if (elect_one()) {
                    issue_scores(tmem + (uint32_t)(t * kRows), qa + (TURNS ? 0 : t * (kTile >> 4)),
                                 ka + (bn % ST) * (kTile >> 4), id_qk);
                    mma_commit(&bars.s_full[t]);
                    if (TURNS || t == ntile - 1) mma_commit(&bars.k_empty[bn % ST]);
                }
                __syncwarp();
            };
            if constexpr (TURNS) {
                scores(n, (int)(n & 1));
                if (nblk > 1) scores(n + 1, (int)(~n & 1));
            } else {
                for (int t = 0; t < ntile; ++t) scores(n, t);
            }
            for (int j = 0; go && j < nblk; ++j, ++n) {
                const uint32_t st = n % ST;
                wait(&bars.v_full[st], n / ST);
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    if (!go || i >= ntile) break;
                    const int t = TURNS ? (int)(n & 1) : i;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        wait(&bars.p_full[t][h], TURNS ? n >> 1 : uses[i] + (uint32_t)j);
                        if (!go) break;
                        if (elect_one()) {
                            const uint32_t o = tmem + (uint32_t)((2 + t) * kRows);
                            const uint32_t pt = tmem + (uint32_t)(t * kRows + h * 64);
                            const uint32_t v = va + st * (kTile >> 4) + h * (8192 >> 4);
#pragma unroll
                            for (int k = 0; k < 4; ++k)  // keys in steps of 16
                                mma_ts(o, pt + 8u * k, desc_of(v + k * (2048 >> 4)), id_pv,
                                       (j >= STEP || h > 0 || k > 0) ? 1u : 0u);
                            if (h == 0) mma_commit(&bars.pv_done[t]);
                            else if (i == ntile - 1) mma_commit(&bars.v_empty[st]);
                        }
                        __syncwarp();
                    }
                    if (go && j + STEP < nblk) scores(n + STEP, t);
                }
            }
            if (elect_one()) mma_commit(&bars.o_full);
            __syncwarp();
#pragma unroll
            for (int t = 0; t < NT; ++t)
                if (t < ntile) uses[t] += (uint32_t)nblk;
            ++seg;
        }
        if (elect_one()) mma_commit(&bars.drain);  // every MMA issued has completed before the CTA can leave
        __syncwarp();
        mbar_wait(&bars.drain, 0, nullptr);
    } else {
        // ---- softmax, one row per thread: warpgroup t has tile t, or every other block (S_t, O_t)
        const int t = warp >> 2, r = tid & (kRows - 1);
        bool got = true;
        uint32_t n0 = 0, seg = 0;                // blocks, segments with keys so far
        uint32_t uses = 0;                       // this tile's blocks so far
        int seq_no = 0;                    // segments
        while (got && walk.next(a, sg)) {
        ++seq_no;
        const int nblk = blocks_of(), ntile = TURNS ? 2 : tiles_of(), first_draft = draft_of(nblk);
        const TreeSeq& w = sg.w;
        const int32_t* bt = a.bt + (int64_t)sg.s * a.bts;
        const int rows = w.n * a.G, trow = sg.rg * NT * kRows + (TURNS ? r : tid), k_begin = sg.k_begin, k_end = sg.k_end;
        const bool live = trow < rows;
        const int tok = live ? trow / a.G : 0;
        const int hq = sg.g * a.G + (live ? trow - tok * a.G : 0);
        const int64_t trow_q = w.q0 + tok;
        T* const orow = reinterpret_cast<T*>(a.out) + trow_q * a.ot + (int64_t)hq * a.oh;
        if (nblk == 0) {  // no key at all
            if (live)
                for (int c = 0; c < kD / 8; ++c) st16(orow + 8 * c, make_uint4(0, 0, 0, 0));
            __syncwarp();
            continue;
        }
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t sS = tmem + lanes + (uint32_t)(t * kRows);
        const uint32_t sO = tmem + lanes + (uint32_t)((2 + t) * kRows);
        const bool idle = !__any_sync(kFull, live);  // none of the warp's rows is one
        const T* qrow = reinterpret_cast<const T*>(a.q) + trow_q * a.qt + (int64_t)hq * a.qh;
        const int64_t* mrow = a.mask + trow_q * a.words;
        float rs = sl2;
        char* const qtile = base + (TURNS ? 0 : t * kTile);
        // the slabs of Q's tile that are this warpgroup's to fill and, at the end, to use for O
        const int slab0 = TURNS ? t : 0, slab1 = TURNS ? t + 1 : 2;
        const int hi = lane >> 3, c = lane & 7, w0 = (warp & 3) * 32;
        {
            // The warp's 32 rows of Q, four at a time (lane: chunk lane % 8 of a slab of row
            // 4 i + lane / 8), into the tile.  (The segment before is done with Q: its O was
            // final, and left through slabs of these rows that this warp alone fills.)
            using P = Packed<T>;
            const int64_t at = live ? trow_q * a.qt + (int64_t)hq * a.qh : -1;
#pragma unroll 1
            for (int sb = slab0; sb < slab1; ++sb)
#pragma unroll 4
                for (int i = 0; i < 8; ++i) {
                    const int64_t o = __shfl_sync(kFull, at, 4 * i + hi);
                    cp_async16_at(smem_u32(qtile) + tile_off(w0 + 4 * i + hi, 8 * sb + c),
                                  reinterpret_cast<const T*>(a.q) + (o < 0 ? 0 : o) + 64 * sb + 8 * c, o < 0 ? 0 : 16);
                }
            cp_async_commit();
            cp_async_wait<0>();
            __syncwarp();
            // rs > 0: a negative scale's sign goes to Q, and 0 becomes as good as 0
            const uint32_t flip = sl2 < 0.f ? 0x80008000u : 0u;
            rs = fabsf(sl2) < 1e-30f ? 1e-30f : fabsf(sl2);
            if (Q8 || flip) {
                // codes: a power-of-two factor brings the row's largest element to [2^14, 2^15)
                int er = 14;  // this thread's own row's exponent
                if constexpr (Q8) {
                    uint32_t top = 0;
#pragma unroll 1
                    for (int sb = slab0; sb < slab1; ++sb)
#pragma unroll 2
                        for (int i = 0; i < 8; ++i) {
                            const uint4 v = *reinterpret_cast<const uint4*>(qtile + tile_off(w0 + 4 * i + hi, 8 * sb + c));
                            uint32_t mx = 0;
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                mx = max(mx, max(__float_as_uint(P::lo(word(v, x))) & 0x7fffffffu,
                                                 __float_as_uint(P::hi(word(v, x))) & 0x7fffffffu));
#pragma unroll
                            for (int o = 4; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(kFull, mx, o));
                            mx = __shfl_sync(kFull, mx, (lane & 3) * 8);  // the thread's row, if it is one of these
                            if ((lane >> 2) == i) top = max(top, mx);
                        }
                    if constexpr (TURNS) {  // the other half of the row is the other warpgroup's
                        qtop[tid] = top;
                        soft_all(true);
                        top = max(top, qtop[tid ^ kRows]);
                    }
                    er = min(max((int)(top >> 23) - 127, -100), 127);
                    rs = fmaxf(rs * __int_as_float((127 - 14 + er) << 23), 1.2e-38f);
                }
#pragma unroll 1
                for (int sb = slab0; sb < slab1; ++sb)
#pragma unroll 2
                    for (int i = 0; i < 8; ++i) {
                        uint4* cell = reinterpret_cast<uint4*>(qtile + tile_off(w0 + 4 * i + hi, 8 * sb + c));
                        uint4 v = *cell;
                        if constexpr (Q8) {
                            const float f = __int_as_float((127 + 14 - __shfl_sync(kFull, er, 4 * i + hi)) << 23);
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                set_word(v, x, MP::pack(P::lo(word(v, x)) * f, P::hi(word(v, x)) * f));
                        }
                        v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
                        *cell = v;
                    }
            }
            proxy_fence();
            mbar_arrive(&bars.q_full);
        }
        float m = -INFINITY, l = 0.f;  // reference maximum and the sum against it
        float unscale = 1.f;           // 2^-x
        for (int j = TURNS ? (int)((t + n0) & 1u) : 0; t < ntile && j < nblk; j += STEP) {
            const uint32_t nb = n0 + (uint32_t)j, phase = TURNS ? nb >> 1 : uses + (uint32_t)j;
            const bool first = j < STEP;
            const int slot = (int)(nb % C::SLOTS), kb = k_begin + j * kRows;
            // what the rows see: over 16-bit rows found while S is on its way (64 trees of 64
            // 348 -> 343 us), over codes, with more to hold, behind it (32 of 32 221 -> 214)
            uint32_t see[4];
            bool masked, near = true;
            auto look = [&]() {
                const uint4 v = *reinterpret_cast<const uint4*>(valid[slot]);
                see[0] = v.x, see[1] = v.y, see[2] = v.z, see[3] = v.w;
                if (j >= first_draft || !live)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        see[q] = live ? see[q] & tree_bits32(mrow, a.words, kb + 32 * q - w.ctx) : 0u;
                masked = __any_sync(kFull, (see[0] & see[1] & see[2] & see[3]) != kFull);
            };
            got = mbar_wait(&bars.info_full[slot], (nb / C::SLOTS) & 1, abort);
            if constexpr (!Q8) look();
            got = got && mbar_wait(&bars.s_full[t], phase & 1, abort);
            if (!__all_sync(kFull, got)) {
                got = false;
                break;
            }
            tc_fence_after();
            if (idle) {  // what is in its rows of P reaches no other row of O
                tc_fence_before();
                mbar_arrive(&bars.p_full[t][0]);
                mbar_arrive(&bars.p_full[t][1]);
                continue;
            }
            if constexpr (Q8) {
                look();
                near = snear[slot] != 0;
                if (first) unscale = __int_as_float((127 - sexp[slot]) << 23);
            }
            // the two halves of a block one after the other: the first's products run during
            // the second's softmax (not unrolled: the roles share the instruction cache)
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
            const int c0 = 64 * h;
            const uint32_t sh = sS + (uint32_t)c0;
            const uint32_t see2[2] = {h ? see[2] : see[0], h ? see[3] : see[1]};
            // The reference moves: O and l with it.
            auto follow = [&](bool move, float to) {
                const float half = move ? ex2(0.5f * (m - to)) : 1.f, corr = half * half;
                if (!first || h > 0) {
                    // O is between two products: those of the block before were done before this
                    // block's S, the first half's are waited for, this half's wait for P
                    if (h == 1) {
                        got = __all_sync(kFull, mbar_wait(&bars.pv_done[t], phase & 1, abort));
                        if (!got) return;
                        tc_fence_after();
                    }
#pragma unroll 1
                    for (int q = 0; q < 4; ++q) {
                        uint32_t o[32];
                        tmem_ld32(sO + 32 * q, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                        tmem_st32(sO + 32 * q, o);
                    }
                }
                l = l * half * half;  // (it may be 2^100 and more where a scale is part of m)
                if (move) m = to;
            };
            if (!Q8 || near) {
            // One pass over S against the reference m, P in registers, the half block's maximum
            // on the side.  While no row's p has grown past 2^TOP (but for the first blocks,
            // nearly always) P stands; else the reference moves, and the pass is made again over
            // S, which P has not touched yet.
            uint32_t pk[32];
            float sum;
            for (int turn = 0;; ++turn) {
                const float mref = m == -INFINITY ? 0.f : m;
                float mx0 = -INFINITY, mx1 = -INFINITY;
                float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
                // the second quarter's load in flight meanwhile, where registers allow
                constexpr int NX = Q8 && NT == 1 ? 1 : 2;
                uint32_t x[NX][32];
                tmem_ld32(sh, x[0]);
                tmem_wait_ld();
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    if (NX == 2 && q == 0) tmem_ld32(sh + 32, x[NX - 1]);
                    uint32_t* xs = x[NX == 2 ? q : 0];
                    const int cq = c0 + 32 * q;
                    if constexpr (Q8) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const float4 k4 = *reinterpret_cast<const float4*>(&sk[slot][cq + e]);
                            float* f = reinterpret_cast<float*>(xs + e);
                            mul2(f[0], f[1], k4.x, k4.y);
                            mul2(f[2], f[3], k4.z, k4.w);
                        }
                    }
                    if (masked) {  // (an unseen key's score may be anything)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!((see2[q] >> e) & 1)) xs[e] = __float_as_uint(-INFINITY);
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        float p[4];
                        // raw maxima: rs > 0 (a negative scale's sign is in Q)
                        mx0 = max3(mx0, __uint_as_float(xs[e]), __uint_as_float(xs[e + 1]));
                        mx1 = max3(mx1, __uint_as_float(xs[e + 2]), __uint_as_float(xs[e + 3]));
                        fma2(p[0], p[1], __uint_as_float(xs[e]), __uint_as_float(xs[e + 1]), rs, -mref);
                        fma2(p[2], p[3], __uint_as_float(xs[e + 2]), __uint_as_float(xs[e + 3]), rs, -mref);
#pragma unroll
                        for (int y = 0; y < 4; ++y) p[y] = ex2(p[y]);
                        add2(s0, s1, p[0], p[1]);
                        add2(s2, s3, p[2], p[3]);
                        if constexpr (Q8) {
                            const float4 v4 = *reinterpret_cast<const float4*>(&sv[slot][cq + e]);
                            mul2(p[0], p[1], v4.x, v4.y);
                            mul2(p[2], p[3], v4.z, v4.w);
                        }
                        pk[16 * q + (e >> 1)] = MP::pack(p[0], p[1]);
                        pk[16 * q + (e >> 1) + 1] = MP::pack(p[2], p[3]);
                    }
                    if (NX == 1 && q == 0) tmem_ld32(sh + 32, x[0]);
                    if (q == 0) tmem_wait_ld();
                }
                sum = (s0 + s1) + (s2 + s3);
                const float mx = fmaxf(mx0, mx1) * rs;
                const bool move = turn == 0 && (mx > m + PR::TOP || (m == -INFINITY && mx > -INFINITY));
                if (!__any_sync(kFull, move)) break;
                follow(move, mx - PR::ROOM);
                if (!got) break;
            }
            if (!got) break;
#pragma unroll
            for (int q = 0; q < 2; ++q) tmem_st16(sh + 16 * q, pk + 16 * q);
            l += sum;
            } else if constexpr (Q8) {
            // V's scales in the exponent, in two passes and small steps (such blocks are rare)
            auto quarter = [&](int c, float mref, float* mx, float* sum, uint32_t* pk) {
                uint32_t x[16];
                tmem_ld16(sh + c, x);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    float u[2], p[2];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const int cc = c + e + y;
                        const bool ok = ((c & 32 ? see2[1] : see2[0]) >> ((c & 31) + e + y)) & 1;
                        const float tt = ok ? __uint_as_float(x[e + y]) * sk[slot][c0 + cc] * rs : -INFINITY;
                        u[y] = ok ? tt + sl[slot][c0 + cc] : -INFINITY;
                        *mx = fmaxf(*mx, tt + fmaxf(sl[slot][c0 + cc], kLeastLog2));
                        *sum += ex2(tt - mref);
                        p[y] = ex2(u[y] - mref);
                    }
                    pk[e >> 1] = MP::pack(p[0], p[1]);
                }
            };
            float mx = -INFINITY, sum = 0.f;
            uint32_t pk[8];
#pragma unroll 1
            for (int c = 0; c < 64; c += 16) quarter(c, 0.f, &mx, &sum, pk);
            const bool move = mx > m + PR::TOP || (m == -INFINITY && mx > -INFINITY);
            if (__any_sync(kFull, move)) follow(move, mx - PR::ROOM);
            if (!got) break;
            sum = 0.f;
#pragma unroll 1
            for (int c = 0; c < 64; c += 16) {
                quarter(c, m == -INFINITY ? 0.f : m, &mx, &sum, pk);
                tmem_st8(sh + c / 2, pk);  // over columns read already
            }
            l += sum;
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bars.p_full[t][h]);
            }
            if (!got) break;
        }
        got = got && mbar_wait(&bars.o_full, seg & 1, abort);
        got = __all_sync(kFull, got);
        const bool whole = sg.slot < 0;
        float own = unscale, other = 0.f;  // what O_t, and the other warpgroup's, are multiplied by
        bool both = false;                 // whether there is the other's
        if constexpr (TURNS) {
            // one row's two sums against the larger reference
            stat[0][tid] = m, stat[1][tid] = l, stat[2][tid] = unscale;
            got = soft_all(got);
            const float m2 = stat[0][tid ^ kRows], top = fmaxf(m, m2);
            const float h = m == -INFINITY ? 0.f : ex2(0.5f * (m - top));
            const float h2 = m2 == -INFINITY ? 0.f : ex2(0.5f * (m2 - top)), f = h * h, f2 = h2 * h2;
            both = nblk > 1;
            own *= f;
            other = stat[2][tid ^ kRows] * f2;
            l = l * h * h + stat[1][tid ^ kRows] * h2 * h2;
            m = top;
        }
        if (whole) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            own *= inv, other *= inv;
        }
        // of one block only one warpgroup has an O
        const uint32_t sA = TURNS && !both ? tmem + lanes + (uint32_t)((2 + (n0 & 1u)) * kRows) : sO;
        const uint32_t sB = tmem + lanes + (uint32_t)((2 + (t ^ 1)) * kRows);
        if (TURNS && !both && (n0 & 1u) != (uint32_t)t) own = other;
        ++seg;
        n0 += (uint32_t)nblk;
        if (t < ntile) uses += (uint32_t)nblk;
        if (got && t < ntile && !idle) {
            tc_fence_after();
            float* part = whole ? nullptr : tree_partial(a, gridDim.x, blockIdx.x, sg.slot, NT * kRows, TURNS ? r : tid, kD);
            // O leaves through Q's tile, which nothing reads any more: each thread its row of a
            // slab there, then the warp's rows, 128 bytes at a time, to memory
            const int64_t to = !live ? -1 : whole ? trow_q * a.ot + (int64_t)hq * a.oh : 0;
            auto leave = [&](int sb, int col) {  // (col: of the row's floats, for partials)
                __syncwarp();
#pragma unroll 4
                for (int i = 0; i < 8; ++i) {
                    const int rr = 4 * i + hi;
                    const int64_t row = __shfl_sync(kFull, to, rr);
                    const uint4 v = *reinterpret_cast<const uint4*>(qtile + tile_off(w0 + rr, 8 * sb + c));
                    if (row >= 0) {
                        if (whole) {
                            st16(reinterpret_cast<T*>(a.out) + row + 64 * sb + 8 * c, v);
                        } else {  // (rows of D + 2 floats: 8-byte aligned)
                            float* dst = tree_partial(a, gridDim.x, blockIdx.x, sg.slot, NT * kRows,
                                                      (TURNS ? 0 : t * kRows) + w0 + rr, kD) + col + 4 * c;
                            *reinterpret_cast<uint2*>(dst) = make_uint2(v.x, v.y);
                            *reinterpret_cast<uint2*>(dst + 2) = make_uint2(v.z, v.w);
                        }
                    }
                }
                __syncwarp();
            };
#pragma unroll 1
            for (int sb = slab0; sb < slab1; ++sb) {
#pragma unroll 1
                for (int q = 0; q < 2; ++q) {
                    float o[32];
                    {
                        uint32_t x[32];
                        tmem_ld32(sA + 64 * sb + 32 * q, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(x[e]) * own;
                        if (TURNS && both) {
                            tmem_ld32(sB + 64 * sb + 32 * q, x);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = fmaf(__uint_as_float(x[e]), other, o[e]);
                        }
                    }
                    if (whole) {
                        using P = Packed<T>;
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            *reinterpret_cast<uint4*>(qtile + tile_off(r, 8 * sb + 4 * q + x)) =
                                make_uint4(P::pack(o[8 * x], o[8 * x + 1]), P::pack(o[8 * x + 2], o[8 * x + 3]),
                                           P::pack(o[8 * x + 4], o[8 * x + 5]), P::pack(o[8 * x + 6], o[8 * x + 7]));
                    } else {
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            *reinterpret_cast<float4*>(qtile + tile_off(r, 8 * sb + x)) =
                                make_float4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
                        leave(sb, 64 * sb + 32 * q);
                    }
                }
                if (whole) leave(sb, 0);
            }
            if (live && !whole && (!TURNS || t == 0)) *reinterpret_cast<float2*>(part + kD) = make_float2(m, l);
            // (set before the last v_full, which o_full follows; the next segment's can only raise
            // it, and makes this one look where nothing is to be found)
            if (live && *static_cast<volatile int*>(&odd_v) >= seq_no) {
                const int j0 = k_begin + min(first_draft, nblk) * kRows;
                if (whole) add_not_finite<T, FMT, T>(a, bt, sg.g, w.ctx, mrow, qrow, sl2, m, j0, k_end, 64 * slab0, 64 * slab1, orow);
                else add_not_finite<T, FMT, float>(a, bt, sg.g, w.ctx, mrow, qrow, sl2, m, j0, k_end, 64 * slab0, 64 * slab1, part);
            }
            __syncwarp();
            tc_fence_before();  // O is read: the next segment's products follow q_full, or p_full
        }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (tid == 0 && abort_flag) flag(a.status, QF_FLAG_TIMEOUT);
    if (warp == C::MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols)
                     : "memory");
    }
}

// A map over a cache (128 dims, B slots, Hkv heads, N blocks): boxes of `box` slots x 64
// dims in the 128-byte swizzle, or x all 128 codes as they are.
bool page_map(CUtensorMap* map, const char* ptr, const TreeDev& a, CUtensorMapDataType type, int box) {
    PFN_cuTensorMapEncodeTiled fn = tensor_map_encode();
    if (!fn || a.N <= 0) return false;
    const cuuint64_t dims[4] = {kD, (cuuint64_t)a.B.d, (cuuint64_t)a.Hkv, (cuuint64_t)a.N};
    const bool codes = type == CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const cuuint64_t es = codes ? 1 : 2;
    const cuuint64_t strides[3] = {(cuuint64_t)a.c2 * es, (cuuint64_t)a.c1 * es, (cuuint64_t)a.c0 * es};
    const cuuint32_t boxes[4] = {codes ? 128u : 64u, (cuuint32_t)box, 1, 1};
    const cuuint32_t step[4] = {1, 1, 1, 1};
    return fn(map, type, 4, const_cast<char*>(ptr), dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
              codes ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int FMT, int NT>
int launch_nt(const TreeDev& a, int ctas, cudaStream_t stream) {
    constexpr auto kernel = tree_tc_kernel<T, FMT, NT>;
    const int rc = allow_smem<kernel>(TreeTc<NT>::SMEM);
    if (rc) return rc;
    // The largest power of two that divides a page and a block: a piece never crosses a
    // page.  Below 8 (the swizzle's rows; codes: 4, a lane per piece), or where the
    // cache's strides make no map, rows come one by one.
    constexpr bool Q8 = FMT != QF_CACHE_PLAIN;
    const CUtensorMapDataType type = Q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                     : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                      : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    CUtensorMap tk{}, tv{};
    int box = std::min(a.B.d & -a.B.d, kRows);
    if (box < (Q8 ? 4 : 8) || !page_map(&tk, a.kc, a, type, box) || !page_map(&tv, a.vc, a, type, box)) box = 0;
    return launch_pdl(kernel, dim3((unsigned)ctas), TreeTc<NT>::THREADS, (size_t)TreeTc<NT>::SMEM, stream, a, tk, tv,
                      box);
}

template <typename T, int FMT>
int launch_fmt(const TreeDev& a, int tiles, int ctas, cudaStream_t stream) {
    return tiles == 1 ? launch_nt<T, FMT, 1>(a, ctas, stream) : launch_nt<T, FMT, 2>(a, ctas, stream);
}

template <typename T>
int launch_t(const TreeDev& a, int format, int tiles, int ctas, cudaStream_t stream) {
    switch (format) {
    case QF_CACHE_PLAIN: return launch_fmt<T, QF_CACHE_PLAIN>(a, tiles, ctas, stream);
    case QF_CACHE_E4M3: return launch_fmt<T, QF_CACHE_E4M3>(a, tiles, ctas, stream);
    default: return launch_fmt<T, QF_CACHE_INT8>(a, tiles, ctas, stream);
    }
}

}  // namespace

int launch_tree_tc(const TreeDev& a, int dtype, int format, int tiles, int ctas, cudaStream_t stream) {
    return dtype == QF_F16 ? launch_t<__half>(a, format, tiles, ctas, stream)
                           : launch_t<__nv_bfloat16>(a, format, tiles, ctas, stream);
}

}  // namespace qf
