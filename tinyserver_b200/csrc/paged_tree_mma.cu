// Paged attention for few query rows per kv head (a decode step's G heads, a
// small tree's tokens x G), 16-bit queries, over a 16-bit or a quantised
// cache.  Bound by HBM: every K and V row is read once and meets at most 16
// rows (8 at head_dim 256).  More rows, at head_dim 64 and 256, where the tcgen05
// kernel has no form, and up to 24 over codes at 128, go in groups of that many, each
// of which reads the keys again, bound by its instructions: 32 trees of 16 and of 64 nodes x 4 heads at 4096 keys, 8 kv heads, over bf16 204 and
// 777 us at head_dim 64, 1495 and 6229 at 256; over e4m3 212 and 749, 775 and 3528.
//
// Warps take tiles of 16 keys in turn, each through a ring of its own in shared
// memory that cp.async fills three or four tiles deep: 40 KB and more per SM in
// flight whatever the registers hold.  The reduction index of a matrix product may
// be permuted as long as both operands agree, and so may the index of its output
// columns, so each lane reads whole 16-byte pieces of rows and calls them the
// fragment elements that mma.sync m16n8k16 wants of it; no transposing loads:
//  * S = Q K^T (rows x keys): B = K^T.  Lane (gid, tig) = (lane / 4, lane % 4)
//    owns keys gid and gid + 8 and, of their rows, 16-byte chunks tig + 4 i; four
//    consecutive elements are its four of one k-step, and Q's fragments are
//    loaded in that same order.
//  * O^T = V^T P^T (dims x rows): A = V^T, B = P^T.  The lane owns the four
//    keys 2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9, whose probabilities the S
//    accumulators already hold in this lane, and 16-byte chunk gid of their
//    rows; a byte permute pairs two keys' elements of one dim.  With the rows
//    as the 8-wide index, 8 rows cost half of what they would as the 16-wide.
// Codes become fp16 in registers (both formats are exact there).  Their row
// scales never touch the codes: K's multiplies the score t, V's enters the
// exponent, p' = 2^(t + log2 vs - m) with m the maximum of that sum (see kLeastLog2), so that p' is
// in [0, 1] however the scales vary; the row's sum takes 2^(t - m), and O / l is the
// definition.  Queries become fp16 after a power-of-two row factor that puts
// their largest element in [2^14, 2^15): exact for every element within 2^-28 of it.
// P goes in as a 16-bit high part and the rounded remainder, so the product
// keeps 16 significant bits or more of p; over codes and for bf16 outputs fp16's 11
// bits, an eighth of the output's own rounding, are enough and the remainder is left
// out.  fp16 ends at 2^-24, so there p is held times 2^15: full precision down to 2^-29
// of a row's largest, and something down to 2^-39.  (Without it 2^18 keys at 2^-25.5, all
// of a row's output beside a key whose V is 0, gave 0.)  Sums and maxima are fp32.
//
// Decode, 4 heads a kv head, 8 kv heads of 128: 256 sequences of up to 8191 keys over
// e4m3 in 416 us (5.5 TB/s); 32 of 2000 keys in 38 us, of 8000 in 106 us: ~15 us besides
// the bytes, a launch each of this kernel and the join's, and per item Q's load, the
// rings' filling and the warps' join.  Issue slots are 54% used over e4m3 (470
// instructions per 16 keys and warp); over bf16 32 of 4096 keys take 101 us (5.3 TB/s).
#include <math.h>

#include "qf_mma.cuh"
#include "qf_quant.cuh"
#include "qf_tree.cuh"

namespace qf {
namespace {

constexpr int kWarps = 4;
constexpr float kRoomLog2 = 15.f;  // P in fp16 is held times 2^15
// In the reference a V scale counts as 2^-100 at least (a row never written has 0): the sum,
// which has no scale in it, grows by 2^100 a key at most, and 2^27 of them stay finite.  Such
// keys' p is below 1 for it: the least scale that the store writes, 2^-108.8, leaves 2^6.2.
constexpr float kLeastLog2 = -100.f;
constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ float pow2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float log2_of(float x) {  // of a normal number
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Whether a word of a V row holds an infinity or a NaN.
template <typename T, int FMT>
__device__ __forceinline__ bool word_not_finite(uint32_t w) {
    if constexpr (FMT == QF_CACHE_E4M3) return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
    else if constexpr (FMT == QF_CACHE_INT8) return false;
    else {
        constexpr uint32_t E = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
        return (w & E) == E || (w & (E << 16)) == (E << 16);
    }
}

template <int FMT, int D>
struct MmaRing {
    static constexpr int EB = FMT == QF_CACHE_PLAIN ? 2 : 1;
    static constexpr int ROW = D * EB;                // bytes per cache row
    static constexpr int NCH = ROW / 16;              // 16-byte chunks per row
    static constexpr int MAT = 16 * ROW;              // one tile of K or V
    static constexpr int STAGE = 2 * MAT + 128 + 16;  // K, V, 16 + 16 scales, valid bits
    static constexpr int STAGES = MAT <= 1024 ? 4 : 3;
    static constexpr int WARP = STAGE * STAGES;
    static constexpr int SMEM = kWarps * WARP;
    // Byte offset of 16-byte chunk c of row r: the rows that a quarter of a warp
    // reads together (r and r + 1 of K, every other one of V) hold one chunk index in
    // different banks.
    __device__ __forceinline__ static int off(int r, int c) {
        const int f = NCH >= 8 ? (r & 6) ^ ((r & 1) << 2) : (r >> 1) & 3;
        return r * ROW + ((c ^ f) << 4);
    }
};

constexpr int kMmaKeys = 16 * kWarps;  // keys of a work unit

// CTAs per SM: by the registers that a kernel needs (wide heads and 16-bit fragments take
// more) and the rings' shared memory.  Decode over e4m3 as above with two, three, four CTAs
// 496, 417, 421 us; of 32 sequences of 8000 keys, 2 kv heads of 8 heads, pages of 64: 41.4,
// 38.8, 41.0; 32 trees of 4 nodes x 4 heads at 4096 keys over e4m3: 92, 85, 137; over bf16,
// one, two: 146, 101; at head_dim 64 over e4m3, three, four, five: 60.4, 59.2, 68.9, of one
// node 46.8, 44.9, 46.1, and over bf16, two, three, four: 55.8, 54.8, 55.3; at head_dim 256
// over e4m3, of one node, one, two: 148, 104.
constexpr int mma_ctas(bool plain, int D) {
    return D == 256 ? (plain ? 1 : 2) : D == 128 ? (plain ? 2 : 3) : plain ? 3 : 4;
}
static_assert(mma_ctas(true, 256) * (MmaRing<QF_CACHE_PLAIN, 256>::SMEM + 2048) <= 233472 &&
                  mma_ctas(false, 256) * (MmaRing<QF_CACHE_E4M3, 256>::SMEM + 2048) <= 233472 &&
                  mma_ctas(true, 128) * (MmaRing<QF_CACHE_PLAIN, 128>::SMEM + 2048) <= 233472 &&
                  mma_ctas(false, 128) * (MmaRing<QF_CACHE_E4M3, 128>::SMEM + 2048) <= 233472 &&
                  mma_ctas(true, 64) * (MmaRing<QF_CACHE_PLAIN, 64>::SMEM + 2048) <= 233472 &&
                  mma_ctas(false, 64) * (MmaRing<QF_CACHE_E4M3, 64>::SMEM + 2048) <= 233472,
              "the rings of an SM's CTAs");

template <typename T, int FMT, int D, int NR>
__global__ void __launch_bounds__(32 * kWarps, mma_ctas(FMT == QF_CACHE_PLAIN, D)) tree_mma_kernel(const TreeDev a) {
    constexpr bool Q8 = FMT != QF_CACHE_PLAIN;
    constexpr bool LO = !Q8 || std::is_same<T, __half>::value;  // P's remainder goes in too
    using MT = typename std::conditional<Q8, __half, T>::type;  // the products' operand type
    using MP = Packed<MT>;
    constexpr float ROOM = std::is_same<MT, __half>::value ? kRoomLog2 : 0.f;
    using R = MmaRing<FMT, D>;
    constexpr int EB = R::EB, ST = R::STAGES;
    constexpr int KS = D / 16;                    // k-steps of Q K^T
    constexpr int NRT = NR / 8;                   // 8-row tiles
    constexpr int KCH = D * EB / 64;              // 16-byte chunks of a K row per lane
    constexpr int VB = D * EB / 8 >= 16 ? 16 : 8;  // bytes per V chunk
    constexpr int VCH = D * EB / 8 / VB;          // V chunks per key and lane
    constexpr int VW = VB / 4;                    // words per V chunk
    constexpr int EPC = VB / EB;                  // dims per V chunk
    constexpr int MTN = D / 16;                   // 16-dim tiles of O^T
    static_assert(kWarps * NR * (D + 2) * 4 <= R::SMEM, "merge area");

    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int scratch[34];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
    const float sl2 = a.scale * 1.4426950408889634f;
    unsigned char* ring = smem + warp * R::WARP;

    pdl_wait();
    pdl_trigger();
    TreeWalk<kMmaKeys, NR, 4> walk;
    walk.begin(a, scratch);
    zero_unowned_rows<T, D>(a);
    if (tid == 0) walk.record(a);

    // a lane's first chunk of a tile within one page, and the way to its next
    const bool one_page = a.B.d % 16 == 0;
    const int64_t lane_off = (int64_t)(lane / R::NCH) * a.c2 * EB + (lane % R::NCH) * 16;
    const int64_t row_step = (int64_t)(32 / R::NCH) * a.c2 * EB;

    TreeSeg sg;
    while (walk.next(a, sg)) {
        const TreeSeq& w = sg.w;
        const int rows = w.n * a.G, r0 = sg.rg * NR, g = sg.g;
        const int32_t* bt = a.bt + (int64_t)sg.s * a.bts;
        const int ntiles = (sg.k_end - sg.k_begin + 15) / 16;  // (0: no key at all)

        // copies of tile i (of this warp: 4 i + warp) into its stage; one group each.  Where
        // pages are multiples of 16 slots a tile lies in one, and its rows are c2 apart.
        int ahead_blk = 0;  // the block of this lane's key of the tile issued next
        auto look = [&](int i) {
            const int j = sg.k_begin + (i * kWarps + warp) * 16 + (lane & 15);
            if (j < sg.k_end) ahead_blk = __ldg(bt + a.B.div(j));
        };
        auto issue = [&](int i) {
            const int j = sg.k_begin + (i * kWarps + warp) * 16 + (lane & 15);
            bool ok = j < sg.k_end;
            const int64_t blk = ahead_blk;
            if (ok && (blk < 0 || blk >= a.N)) {
                flag(a.status, QF_FLAG_BAD_BLOCK);
                ok = false;
            }
            const int slot = j - a.B.div(j) * a.B.d;
            const int64_t row = ok ? (blk * a.c0 + (int64_t)g * a.c1 + (int64_t)slot * a.c2) * EB : 0;
            const int64_t srow = Q8 && ok ? blk * a.s0 + (int64_t)g * a.s1 + (int64_t)slot * a.s2 : 0;
            look(i + 1);
            const unsigned valid = __ballot_sync(kAll, ok) & 0xffffu;
            unsigned char* kt = ring + (i % ST) * R::STAGE;
            unsigned char* vt = kt + R::MAT;
            if (valid == 0xffffu && one_page) {
                const int64_t first = __shfl_sync(kAll, row, 0) + lane_off;
#pragma unroll
                for (int x = 0; x < R::NCH / 2; ++x) {
                    const int r = (x * 32 + lane) / R::NCH, c = (x * 32 + lane) % R::NCH;
                    const int64_t o = first + x * row_step;
                    cp_async16(kt + R::off(r, c), a.kc + o, 16);
                    cp_async16(vt + R::off(r, c), a.vc + o, 16);
                }
            } else if (valid) {
#pragma unroll 2
                for (int x = 0; x < R::NCH / 2; ++x) {
                    const int idx = x * 32 + lane, r = idx / R::NCH, c = idx % R::NCH;
                    const int64_t o = __shfl_sync(kAll, row, r);
                    const int bytes = (valid >> r) & 1 ? 16 : 0;
                    cp_async16(kt + R::off(r, c), a.kc + o + c * 16, bytes);
                    cp_async16(vt + R::off(r, c), a.vc + o + c * 16, bytes);
                }
            }
            if (Q8 && ok)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(static_cast<uint32_t>(
                                 __cvta_generic_to_shared(kt + 2 * R::MAT + lane * 4))),
                             "l"((lane < 16 ? a.ks : a.vs) + srow)
                             : "memory");
            if (lane == 0) *reinterpret_cast<unsigned*>(kt + 2 * R::MAT + 128) = valid;
            cp_async_commit();
        };
        look(0);
#pragma unroll
        for (int i = 0; i < ST - 1; ++i) issue(i);

        // Q fragments, rows gid and gid + 8 of the tile, four consecutive dims per k-step
        uint32_t qa[KS][2 * NRT];
        float rs[NRT];  // what a row's products are multiplied by
        const int64_t* mrow[NRT];
#pragma unroll
        for (int nt = 0; nt < NRT; ++nt) {
            const int r = r0 + nt * 8 + gid, tok = r / a.G;
            const bool live = r < rows;
            const char* qp = a.q + ((int64_t)(w.q0 + (live ? tok : 0)) * a.qt +
                                    (int64_t)(g * a.G + (live ? r - tok * a.G : 0)) * a.qh) * 2;
            mrow[nt] = a.mask + (int64_t)(w.q0 + (live ? tok : 0)) * a.words;
            uint2 raw[KS];
            uint32_t mx = 0;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d = Q8 ? (ks >> 2) * 64 + tig * 16 + (ks & 3) * 4
                                 : (ks >> 1) * 32 + tig * 8 + (ks & 1) * 4;
                raw[ks] = live ? __ldg(reinterpret_cast<const uint2*>(qp + d * 2)) : make_uint2(0, 0);
                if constexpr (Q8) {
                    using P = Packed<T>;
                    mx = max(max(mx, __float_as_uint(P::lo(raw[ks].x)) & 0x7fffffffu),
                             __float_as_uint(P::hi(raw[ks].x)) & 0x7fffffffu);
                    mx = max(max(mx, __float_as_uint(P::lo(raw[ks].y)) & 0x7fffffffu),
                             __float_as_uint(P::hi(raw[ks].y)) & 0x7fffffffu);
                }
            }
            rs[nt] = sl2;
            float f = 1.f;
            if constexpr (Q8) {
                mx = max(mx, __shfl_xor_sync(kAll, mx, 1));
                mx = max(mx, __shfl_xor_sync(kAll, mx, 2));
                // largest element's exponent e: factor 2^(14 - e), its inverse with the scores
                const int e = min(max((int)(mx >> 23) - 127, -100), 127);
                f = __int_as_float((127 + 14 - e) << 23);
                rs[nt] = sl2 * __int_as_float((127 - 14 + e) << 23);
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if constexpr (Q8) {
                    using P = Packed<T>;
                    qa[ks][nt] = MP::pack(P::lo(raw[ks].x) * f, P::hi(raw[ks].x) * f);
                    qa[ks][NRT + nt] = MP::pack(P::lo(raw[ks].y) * f, P::hi(raw[ks].y) * f);
                } else {
                    qa[ks][nt] = raw[ks].x;
                    qa[ks][NRT + nt] = raw[ks].y;
                }
            }
        }

        float acc[NRT][MTN][4];
        float m[NRT], l[NRT];  // reference: max of t (+ log2 v-scale); this lane's sum against it
#pragma unroll
        for (int nt = 0; nt < NRT; ++nt) {
            m[nt] = -INFINITY;
            l[nt] = 0.f;
#pragma unroll
            for (int i = 0; i < MTN; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
        }

        for (int i = 0; i * kWarps + warp < ntiles; ++i) {
            issue(i + ST - 1);
            cp_async_wait<ST - 1>();
            __syncwarp();
            const int j0 = sg.k_begin + (i * kWarps + warp) * 16;
            const unsigned char* kt = ring + (i % ST) * R::STAGE;
            const unsigned char* vt = kt + R::MAT;
            const unsigned valid = *reinterpret_cast<const unsigned*>(kt + 2 * R::MAT + 128);
            if (valid) {
                // S = Q K^T
                float sc[2][4];
#pragma unroll
                for (int n = 0; n < 2; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
                for (int c = 0; c < KCH; ++c) {
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const uint4 kf = *reinterpret_cast<const uint4*>(kt + R::off(n * 8 + gid, tig + 4 * c));
#pragma unroll
                        for (int x = 0; x < (Q8 ? 4 : 2); ++x) {
                            const int ks = c * (Q8 ? 4 : 2) + x;
                            uint32_t b0, b1;
                            if constexpr (Q8) codes_to_f16<FMT>(word(kf, x), b0, b1);
                            else b0 = word(kf, 2 * x), b1 = word(kf, 2 * x + 1);
                            const uint32_t fr[4] = {qa[ks][0], NRT == 2 ? qa[ks][1] : 0u, qa[ks][NRT],
                                                    NRT == 2 ? qa[ks][2 * NRT - 1] : 0u};
                            Mma<MT>::run(sc[n], fr, b0, b1);
                        }
                    }
                }

                // online softmax; this lane: rows gid (+ 8), keys 8 n + 2 tig + e
                const bool draft = a.cu && j0 + 16 > w.ctx;
                float ksv[2][2], lvv[2][2];  // K's scales, log2 of V's (-inf: a scale of 0, values of 0)
                if constexpr (Q8) {
                    const float* sp = reinterpret_cast<const float*>(kt + 2 * R::MAT);
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const float2 k2 = *reinterpret_cast<const float2*>(sp + 8 * n + 2 * tig);
                        const float2 v2 = *reinterpret_cast<const float2*>(sp + 16 + 8 * n + 2 * tig);
                        ksv[n][0] = k2.x, ksv[n][1] = k2.y;
                        lvv[n][0] = log2_of(v2.x);
                        lvv[n][1] = log2_of(v2.y);
                    }
                }
                float pw[NRT][2][2];
                unsigned seen[NRT];
                uint32_t ph[NRT][2], pl[NRT][2];
                float corr[NRT];
                bool moved = false;
#pragma unroll
                for (int nt = 0; nt < NRT; ++nt) {
                    seen[nt] = valid;
                    if (draft) seen[nt] &= tree_bits32(mrow[nt], a.words, j0 - w.ctx);
                    float t[2][2], u[2][2], mx = -INFINITY;
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const bool ok = (seen[nt] >> (8 * n + 2 * tig + e)) & 1;
                            float x = sc[n][2 * nt + e] * rs[nt];
                            if constexpr (Q8) x *= ksv[n][e];
                            t[n][e] = ok ? x : -INFINITY;
                            u[n][e] = Q8 ? (ok ? x + lvv[n][e] : -INFINITY) : t[n][e];
                            mx = fmaxf(mx, Q8 ? t[n][e] + fmaxf(lvv[n][e], kLeastLog2) : t[n][e]);
                        }
                    mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 2));
                    const float mn = fmaxf(m[nt], mx), base = mn == -INFINITY ? 0.f : mn;
                    // (in two steps: l may be 2^100 and more, see kLeastLog2, and what is left
                    // of it count, where the factor alone is too small for a float)
                    const float half = pow2(0.5f * (m[nt] - base));
                    corr[nt] = half * half;
                    m[nt] = mn;
                    const float pbase = base - ROOM;
                    float sum = 0.f;  // (over codes of p itself, else of p times 2^ROOM)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            pw[nt][n][e] = pow2(u[n][e] - pbase);
                            sum += Q8 ? pow2(t[n][e] - base) : pw[nt][n][e];
                        }
                    l[nt] = l[nt] * half * half + sum;
                    moved |= corr[nt] != 1.f;
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        ph[nt][n] = MP::pack(pw[nt][n][0], pw[nt][n][1]);
                        if (LO) pl[nt][n] = MP::pack(pw[nt][n][0] - MP::lo(ph[nt][n]), pw[nt][n][1] - MP::hi(ph[nt][n]));
                    }
                }
                if (__any_sync(kAll, moved)) {
#pragma unroll
                    for (int nt = 0; nt < NRT; ++nt) {
                        const float c0 = __shfl_sync(kAll, corr[nt], 8 * tig);
                        const float c1 = __shfl_sync(kAll, corr[nt], 8 * tig + 4);
#pragma unroll
                        for (int x = 0; x < MTN; ++x) {
                            acc[nt][x][0] *= c0;
                            acc[nt][x][1] *= c1;
                            acc[nt][x][2] *= c0;
                            acc[nt][x][3] *= c1;
                        }
                    }
                }

                // V rows of keys 2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9
                uint32_t vf[4][VCH][VW];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int k = 2 * tig + (x & 1) + (x >> 1) * 8;
#pragma unroll
                    for (int c = 0; c < VCH; ++c) {
                        if constexpr (VB == 16) {
                            const uint4 v = *reinterpret_cast<const uint4*>(vt + R::off(k, gid + 8 * c));
                            vf[x][c][0] = v.x, vf[x][c][1] = v.y, vf[x][c][2] = v.z, vf[x][c][3] = v.w;
                        } else {
                            const uint2 v = *reinterpret_cast<const uint2*>(vt + R::off(k, gid >> 1) + (gid & 1) * 8);
                            vf[x][c][0] = v.x, vf[x][c][1] = v.y;
                        }
                    }
                }
                // An infinity or a NaN in the V of a drafted key that some row does not
                // see: 0 times it is not 0, so such a (rare) tile is added up key by key,
                // a row's unseen keys left out.
                bool odd = false;
                if (draft) {
#pragma unroll
                    for (int x = 0; x < 4; ++x)
#pragma unroll
                        for (int c = 0; c < VCH; ++c)
#pragma unroll
                            for (int y = 0; y < VW; ++y) odd |= word_not_finite<T, FMT>(vf[x][c][y]);
                    odd = __any_sync(kAll, odd);
                }
                if (odd) {
                    for (int k = 0; k < 16; ++k) {
                        float pr[NRT][2];
                        bool in[NRT][2];
#pragma unroll
                        for (int nt = 0; nt < NRT; ++nt) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {  // rows 2 tig + e: lanes 4 (2 tig + e) + key pair
                                const int from = 4 * (2 * tig + e) + ((k & 7) >> 1);
                                const float x0 = __shfl_sync(kAll, pw[nt][0][0], from);
                                const float x1 = __shfl_sync(kAll, pw[nt][0][1], from);
                                const float x2 = __shfl_sync(kAll, pw[nt][1][0], from);
                                const float x3 = __shfl_sync(kAll, pw[nt][1][1], from);
                                pr[nt][e] = k < 8 ? (k & 1 ? x1 : x0) : (k & 1 ? x3 : x2);
                                in[nt][e] = (__shfl_sync(kAll, seen[nt], from) >> k) & 1;
                            }
                        }
#pragma unroll
                        for (int x = 0; x < MTN; ++x) {
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                const int d = (x / (EPC / 2)) * (EPC * 8) + gid * EPC + 2 * (x % (EPC / 2)) + half;
                                const unsigned char* at = vt + R::off(k, d * EB / 16) + (d * EB & 15);
                                float v;
                                if constexpr (Q8) v = code_to_float<FMT>(*at);
                                else v = Dt<T>::to_f(*reinterpret_cast<const T*>(at));
#pragma unroll
                                for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
                                    for (int e = 0; e < 2; ++e)
                                        if (in[nt][e])
                                            acc[nt][x][2 * half + e] = fmaf(pr[nt][e], v, acc[nt][x][2 * half + e]);
                            }
                        }
                    }
                } else {
                    // O^T += V^T P^T
#pragma unroll
                    for (int c = 0; c < VCH; ++c) {
#pragma unroll
                        for (int x = 0; x < VW; ++x) {
#pragma unroll
                            for (int half = 0; half < (Q8 ? 2 : 1); ++half) {
                                uint32_t va[4];
                                if constexpr (Q8) {
                                    const uint32_t sel = half ? 0x7362u : 0x5140u;
                                    codes_to_f16<FMT>(__byte_perm(vf[0][c][x], vf[1][c][x], sel), va[0], va[1]);
                                    codes_to_f16<FMT>(__byte_perm(vf[2][c][x], vf[3][c][x], sel), va[2], va[3]);
                                } else {
                                    va[0] = __byte_perm(vf[0][c][x], vf[1][c][x], 0x5410);
                                    va[1] = __byte_perm(vf[0][c][x], vf[1][c][x], 0x7632);
                                    va[2] = __byte_perm(vf[2][c][x], vf[3][c][x], 0x5410);
                                    va[3] = __byte_perm(vf[2][c][x], vf[3][c][x], 0x7632);
                                }
                                const int y = c * (EPC / 2) + (Q8 ? 2 * x + half : x);
#pragma unroll
                                for (int nt = 0; nt < NRT; ++nt) {
                                    Mma<MT>::run(acc[nt][y], va, ph[nt][0], ph[nt][1]);
                                    if (LO) Mma<MT>::run(acc[nt][y], va, pl[nt][0], pl[nt][1]);
                                }
                            }
                        }
                    }
                }
            }
            __syncwarp();  // every lane is done with this stage before it is refilled
        }
        cp_async_wait<0>();
        __syncthreads();  // the rings become the merge area

        float* wm = reinterpret_cast<float*>(smem);  // [warps][NR] maxima, sums, then [warps][NR][D]
        float* wl = wm + kWarps * NR;
        float* wacc = wl + kWarps * NR;
#pragma unroll
        for (int nt = 0; nt < NRT; ++nt) {
            l[nt] += __shfl_xor_sync(kAll, l[nt], 1);
            l[nt] += __shfl_xor_sync(kAll, l[nt], 2);
            if (tig == 0) {
                wm[warp * NR + nt * 8 + gid] = m[nt];
                wl[warp * NR + nt * 8 + gid] = l[nt];
            }
#pragma unroll
            for (int x = 0; x < MTN; ++x) {
                const int d = (x / (EPC / 2)) * (EPC * 8) + gid * EPC + 2 * (x % (EPC / 2));
                float* at = wacc + (warp * NR + nt * 8 + 2 * tig) * D + d;
                *reinterpret_cast<float2*>(at) = make_float2(acc[nt][x][0], acc[nt][x][2]);
                *reinterpret_cast<float2*>(at + D) = make_float2(acc[nt][x][1], acc[nt][x][3]);
            }
        }
        __syncthreads();
        for (int i = tid; i < NR * D; i += 32 * kWarps) {
            const int ri = i / D, d = i % D, r = r0 + ri;
            if (r >= rows) break;
            float M = -INFINITY, Ls = 0.f, A = 0.f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) M = fmaxf(M, wm[k * NR + ri]);
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                const float f = M == -INFINITY ? 0.f : exp2f(0.5f * (wm[k * NR + ri] - M));  // its half
                Ls += wl[k * NR + ri] * f * f;
                A += wacc[(k * NR + ri) * D + d] * f * f;
            }
            if constexpr (Q8) A *= 1.f / (1 << (int)kRoomLog2);
            if (sg.slot < 0) {
                // (no weight at all: 0, or NaN where every key the row sees has a NaN for a scale)
                const int tok = r / a.G;
                reinterpret_cast<T*>(a.out)[(int64_t)(w.q0 + tok) * a.ot + (int64_t)(g * a.G + r - tok * a.G) * a.oh + d] =
                    Dt<T>::from_f(Ls == 0.f ? A * 0.f : A / Ls);
            } else {
                float* o = tree_partial(a, gridDim.x, blockIdx.x, sg.slot, NR, ri, D);
                o[d] = A;
                if (d == 0) {
                    o[D] = M;
                    o[D + 1] = Ls;
                }
            }
        }
        __syncthreads();  // the merge area becomes the rings again
    }
}

template <typename T, int FMT, int D, int NR>
int launch_nr(const TreeDev& a, int ctas, cudaStream_t stream) {
    constexpr auto kernel = tree_mma_kernel<T, FMT, D, NR>;
    const int rc = allow_smem<kernel>(MmaRing<FMT, D>::SMEM);
    if (rc) return rc;
    return launch_pdl(kernel, dim3((unsigned)ctas), 32 * kWarps, (size_t)MmaRing<FMT, D>::SMEM, stream, a);
}

template <typename T, int FMT>
int launch_d(const TreeDev& a, int D, int rows, int ctas, cudaStream_t stream) {
    switch (D) {
    case 64:
        return rows == 8 ? launch_nr<T, FMT, 64, 8>(a, ctas, stream) : launch_nr<T, FMT, 64, 16>(a, ctas, stream);
    case 128:
        return rows == 8 ? launch_nr<T, FMT, 128, 8>(a, ctas, stream) : launch_nr<T, FMT, 128, 16>(a, ctas, stream);
    default:  // 16 rows of 256 would not fit the registers
        return launch_nr<T, FMT, 256, 8>(a, ctas, stream);
    }
}

template <typename T>
int launch_fmt(const TreeDev& a, int format, int D, int rows, int ctas, cudaStream_t stream) {
    switch (format) {
    case QF_CACHE_PLAIN: return launch_d<T, QF_CACHE_PLAIN>(a, D, rows, ctas, stream);
    case QF_CACHE_E4M3: return launch_d<T, QF_CACHE_E4M3>(a, D, rows, ctas, stream);
    default: return launch_d<T, QF_CACHE_INT8>(a, D, rows, ctas, stream);
    }
}

}  // namespace

int tree_mma_ctas_per_sm(bool plain, int D) { return mma_ctas(plain, D); }

int launch_tree_mma(const TreeDev& a, int dtype, int format, int D, int rows, int ctas,
                    cudaStream_t stream) {
    return dtype == QF_F16 ? launch_fmt<__half>(a, format, D, rows, ctas, stream)
                           : launch_fmt<__nv_bfloat16>(a, format, D, rows, ctas, stream);
}

}  // namespace qf
