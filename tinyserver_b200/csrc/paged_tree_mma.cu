// Paged attention for few query rows per kv head (a decode step's G heads, a
// small tree's tokens x G), 16-bit queries, over a 16-bit or a quantised
// cache.  Bound by HBM: every K and V row is read once and meets at most 16
// rows.
//
// Warps take tiles of 16 keys in turn; nothing of K or V passes through shared
// memory.  The reduction index of a matrix product may be permuted as long as
// both operands agree, and so may the index of its output columns, so each
// lane loads whole 16-byte pieces of rows and calls them the fragment
// elements that mma.sync m16n8k16 wants of it:
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
// scales never touch the codes: K's multiplies the score, V's enters the
// exponent, p' = 2^(t + log2 scale - m'), with a running maximum m' of its own,
// so that p' is in [0, 1] however the scales vary.  Queries become fp16 after a
// power-of-two row factor that puts their largest element in [2^14, 2^15): exact
// for every element within 2^-28 of it.
// P goes in as a 16-bit high part and the rounded remainder, so the product
// keeps 16 significant bits or more of p; sums and maxima are fp32.
//
// Per warp one K tile is in flight while the one before is multiplied, and V is
// issued before QK: 8 to 12 resident warps keep 40 KB or more per SM in flight.
#include <math.h>

#include "qf_mma.cuh"
#include "qf_quant.cuh"
#include "qf_tree.cuh"

namespace qf {
namespace {

constexpr int kWarps = 4;
constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ float pow2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

template <typename T, int FMT, int D, int NR>
__global__ void __launch_bounds__(32 * kWarps) tree_mma_kernel(const TreeDev a) {
    constexpr bool Q8 = FMT != QF_CACHE_PLAIN;
    using MT = typename std::conditional<Q8, __half, T>::type;  // the products' operand type
    using MP = Packed<MT>;
    constexpr int EB = Q8 ? 1 : 2;                // bytes per cache element
    constexpr int KS = D / 16;                    // k-steps of Q K^T
    constexpr int NRT = NR / 8;                   // 8-row tiles
    constexpr int KCH = D * EB / 64;              // 16-byte chunks of a K row per lane
    constexpr int VB = D * EB / 8 >= 16 ? 16 : 8;  // bytes per V chunk
    constexpr int VCH = D * EB / 8 / VB;          // V chunks per key and lane
    constexpr int VW = VB / 4;                    // words per V chunk
    constexpr int EPC = VB / EB;                  // dims per V chunk
    constexpr int MTN = D / 16;                   // 16-dim tiles of O^T

    const int p = blockIdx.x, s = blockIdx.z;
    const int g = blockIdx.y % a.Hkv, rg = blockIdx.y / a.Hkv;
    const TreeSeq w = tree_seq(a, s);
    if (p == 0 && rg == 0) zero_unowned_rows<T, D>(a, s, g, w);
    const int rows = w.n * a.G, r0 = rg * NR;
    if (p >= w.nparts || r0 >= rows) return;
    const int k_begin = p * a.part, k_end = k_begin + min(w.L - k_begin, a.part);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
    const int32_t* bt = a.bt + (int64_t)s * a.bts;
    const float sl2 = a.scale * 1.4426950408889634f;

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
    float m[NRT], mo[NRT], l[NRT];  // max of t, max of t + log2 v-scale, this lane's sum
#pragma unroll
    for (int nt = 0; nt < NRT; ++nt) {
        m[nt] = mo[nt] = -INFINITY;
        l[nt] = 0.f;
#pragma unroll
        for (int i = 0; i < MTN; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
    }

    // lane k < 16: where key j0 + k is, and its scales; the tile's valid keys as a mask
    struct Tile {
        int64_t row;
        float ks, lv;
        unsigned valid;
    };
    auto locate = [&](int j0) {
        Tile t{0, 0.f, 0.f, 0u};
        bool ok = false;
        int64_t srow = 0;
        if (lane < 16 && j0 + lane < k_end) ok = key_place(a, bt, g, j0 + lane, t.row, srow);
        if (Q8 && ok) {
            t.ks = __ldg(a.ks + srow);
            t.lv = __log2f(__ldg(a.vs + srow));
        }
        t.valid = __ballot_sync(kAll, ok);
        return t;
    };
    uint4 kf[2][KCH];
    auto load_k = [&](const Tile& t) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int64_t row = __shfl_sync(kAll, t.row, n * 8 + gid);
            const bool ok = (t.valid >> (n * 8 + gid)) & 1;
#pragma unroll
            for (int i = 0; i < KCH; ++i)
                kf[n][i] = ok ? ld_stream16(a.kc + row * EB + i * 64 + tig * 16) : make_uint4(0, 0, 0, 0);
        }
    };

    int j0 = k_begin + warp * 16;
    Tile cur = locate(j0);  // (no key at all: an empty mask, no loads)
    load_k(cur);
    for (; j0 < k_end; j0 += kWarps * 16) {
        // V rows of keys 2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9
        uint32_t vf[4][VCH][VW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = 2 * tig + (i & 1) + (i >> 1) * 8;
            const int64_t row = __shfl_sync(kAll, cur.row, k);
            const bool ok = (cur.valid >> k) & 1;
#pragma unroll
            for (int c = 0; c < VCH; ++c) {
                const char* vp = a.vc + row * EB + c * 128 + gid * VB;
                if constexpr (VB == 16) {
                    const uint4 v = ok ? ld_stream16(vp) : make_uint4(0, 0, 0, 0);
                    vf[i][c][0] = v.x, vf[i][c][1] = v.y, vf[i][c][2] = v.z, vf[i][c][3] = v.w;
                } else {
                    const uint2 v = ok ? ld_stream8(vp) : make_uint2(0, 0);
                    vf[i][c][0] = v.x, vf[i][c][1] = v.y;
                }
            }
        }
        Tile next = locate(j0 + kWarps * 16);

        // S = Q K^T
        float sc[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
        for (int i = 0; i < KCH; ++i) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
#pragma unroll
                for (int x = 0; x < (Q8 ? 4 : 2); ++x) {
                    const int ks = i * (Q8 ? 4 : 2) + x;
                    uint32_t b0, b1;
                    if constexpr (Q8) codes_to_f16<FMT>(word(kf[n][i], x), b0, b1);
                    else b0 = word(kf[n][i], 2 * x), b1 = word(kf[n][i], 2 * x + 1);
                    const uint32_t fr[4] = {qa[ks][0], NRT == 2 ? qa[ks][1] : 0u, qa[ks][NRT],
                                            NRT == 2 ? qa[ks][2 * NRT - 1] : 0u};
                    Mma<MT>::run(sc[n], fr, b0, b1);
                }
            }
        }
        load_k(next);

        // online softmax; this lane: rows gid (+ 8), keys 8 n + 2 tig + e
        const bool draft = a.cu && j0 + 16 > w.ctx;
        float ksv[2][2], lvv[2][2];
        if constexpr (Q8) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    ksv[n][e] = __shfl_sync(kAll, cur.ks, 8 * n + 2 * tig + e);
                    lvv[n][e] = __shfl_sync(kAll, cur.lv, 8 * n + 2 * tig + e);
                }
        }
        float pw[NRT][2][2];
        unsigned seen[NRT];
        uint32_t ph[NRT][2], pl[NRT][2];
        float corr[NRT];
        bool moved = false;
#pragma unroll
        for (int nt = 0; nt < NRT; ++nt) {
            seen[nt] = cur.valid;
            if (draft) seen[nt] &= tree_bits32(mrow[nt], a.words, j0 - w.ctx);
            float t[2][2], u[2][2], mx = -INFINITY, mu = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool ok = (seen[nt] >> (8 * n + 2 * tig + e)) & 1;
                    float x = sc[n][2 * nt + e] * rs[nt];
                    if constexpr (Q8) x *= ksv[n][e];
                    t[n][e] = ok ? x : -INFINITY;
                    mx = fmaxf(mx, t[n][e]);
                    if constexpr (Q8) {
                        u[n][e] = ok ? x + lvv[n][e] : -INFINITY;
                        mu = fmaxf(mu, u[n][e]);
                    }
                }
            mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 2));
            const float mn = fmaxf(m[nt], mx), base = mn == -INFINITY ? 0.f : mn;
            const float cl = pow2(m[nt] - base);
            m[nt] = mn;
            corr[nt] = cl;
            float sum = 0.f, obase = base;
            if constexpr (Q8) {
                mu = fmaxf(mu, __shfl_xor_sync(kAll, mu, 1));
                mu = fmaxf(mu, __shfl_xor_sync(kAll, mu, 2));
                const float un = fmaxf(mo[nt], mu);
                obase = un == -INFINITY ? 0.f : un;
                corr[nt] = pow2(mo[nt] - obase);
                mo[nt] = un;
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float pr = pow2(t[n][e] - base);
                    sum += pr;
                    pw[nt][n][e] = Q8 ? pow2(u[n][e] - obase) : pr;
                }
            l[nt] = l[nt] * cl + sum;
            moved |= corr[nt] != 1.f;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                ph[nt][n] = MP::pack(pw[nt][n][0], pw[nt][n][1]);
                pl[nt][n] = MP::pack(pw[nt][n][0] - MP::lo(ph[nt][n]), pw[nt][n][1] - MP::hi(ph[nt][n]));
            }
        }
        if (__any_sync(kAll, moved)) {
#pragma unroll
            for (int nt = 0; nt < NRT; ++nt) {
                const float c0 = __shfl_sync(kAll, corr[nt], 8 * tig);
                const float c1 = __shfl_sync(kAll, corr[nt], 8 * tig + 4);
#pragma unroll
                for (int i = 0; i < MTN; ++i) {
                    acc[nt][i][0] *= c0;
                    acc[nt][i][1] *= c1;
                    acc[nt][i][2] *= c0;
                    acc[nt][i][3] *= c1;
                }
            }
        }

        // An infinity or a NaN in the V of a drafted key that some row does not
        // see: 0 times it is not 0, so such a (rare) tile is added up key by key,
        // a row's unseen keys left out.
        bool odd = false;
        if (draft) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < VCH; ++c)
#pragma unroll
                    for (int x = 0; x < VW; ++x) odd |= word_not_finite<T, FMT>(vf[i][c][x]);
            odd = __any_sync(kAll, odd);
        }
        if (odd) {
            for (int k = 0; k < 16; ++k) {
                const int64_t row = __shfl_sync(kAll, cur.row, k);
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
                if (!((cur.valid >> k) & 1)) continue;
#pragma unroll
                for (int i = 0; i < MTN; ++i) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int d = (i / (EPC / 2)) * (EPC * 8) + gid * EPC + 2 * (i % (EPC / 2)) + half;
                        float v;
                        if constexpr (Q8) v = code_to_float<FMT>(reinterpret_cast<const uint8_t*>(a.vc)[row + d]);
                        else v = Dt<T>::to_f(reinterpret_cast<const T*>(a.vc)[row + d]);
#pragma unroll
                        for (int nt = 0; nt < NRT; ++nt)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if (in[nt][e]) acc[nt][i][2 * half + e] = fmaf(pr[nt][e], v, acc[nt][i][2 * half + e]);
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
                        const int i = c * (EPC / 2) + (Q8 ? 2 * x + half : x);
#pragma unroll
                        for (int nt = 0; nt < NRT; ++nt) {
                            Mma<MT>::run(acc[nt][i], va, ph[nt][0], ph[nt][1]);
                            Mma<MT>::run(acc[nt][i], va, pl[nt][0], pl[nt][1]);
                        }
                    }
                }
            }
        }
        cur = next;
    }

    // merge the warps through shared memory
    __shared__ float wm[kWarps][NR], wl[kWarps][NR];
    __shared__ __align__(16) float wacc[kWarps][NR][D];
#pragma unroll
    for (int nt = 0; nt < NRT; ++nt) {
        l[nt] += __shfl_xor_sync(kAll, l[nt], 1);
        l[nt] += __shfl_xor_sync(kAll, l[nt], 2);
        if (tig == 0) {
            wm[warp][nt * 8 + gid] = m[nt];
            wl[warp][nt * 8 + gid] = l[nt];
        }
        // accumulators against m' (scales in) brought back against m
        const float f = Q8 ? (m[nt] == -INFINITY ? 0.f : exp2f(mo[nt] - m[nt])) : 1.f;
        const float f0 = __shfl_sync(kAll, f, 8 * tig), f1 = __shfl_sync(kAll, f, 8 * tig + 4);
#pragma unroll
        for (int i = 0; i < MTN; ++i) {
            const int d = (i / (EPC / 2)) * (EPC * 8) + gid * EPC + 2 * (i % (EPC / 2));
            *reinterpret_cast<float2*>(&wacc[warp][nt * 8 + 2 * tig][d]) =
                make_float2(acc[nt][i][0] * f0, acc[nt][i][2] * f0);
            *reinterpret_cast<float2*>(&wacc[warp][nt * 8 + 2 * tig + 1][d]) =
                make_float2(acc[nt][i][1] * f1, acc[nt][i][3] * f1);
        }
    }
    __syncthreads();
    for (int i = tid; i < NR * D; i += 32 * kWarps) {
        const int ri = i / D, d = i % D, r = r0 + ri;
        if (r >= rows) break;
        float M = -INFINITY, Ls = 0.f, A = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) M = fmaxf(M, wm[k][ri]);
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            const float f = M == -INFINITY ? 0.f : exp2f(wm[k][ri] - M);
            Ls += wl[k][ri] * f;
            A += wacc[k][ri][d] * f;
        }
        const int tok = r / a.G;
        const int64_t t = w.q0 + tok, h = g * a.G + (r - tok * a.G);
        if (w.nparts == 1) {
            reinterpret_cast<T*>(a.out)[t * a.ot + h * a.oh + d] =
                Dt<T>::from_f(Ls == 0.f ? 0.f : A / Ls);
        } else {
            float* o = a.ws + ((t * a.Hq + h) * a.P + p) * (D + 2);
            o[d] = A;
            if (d == 0) {
                o[D] = M;
                o[D + 1] = Ls;
            }
        }
    }
}

template <typename T, int FMT, int D, int NR>
int launch_nr(const TreeDev& a, int rows, cudaStream_t stream) {
    const int64_t groups = ceil_div(rows, NR);
    if (groups * a.Hkv > 65535) return QF_ERR_UNSUPPORTED;
    tree_mma_kernel<T, FMT, D, NR><<<dim3((unsigned)a.P, (unsigned)(groups * a.Hkv), (unsigned)a.S),
                                     32 * kWarps, 0, stream>>>(a);
    return check_launch();
}

template <typename T, int FMT>
int launch_d(const TreeDev& a, int D, int rows, cudaStream_t stream) {
    switch (D) {
    case 64:
        return rows <= 8 ? launch_nr<T, FMT, 64, 8>(a, rows, stream) : launch_nr<T, FMT, 64, 16>(a, rows, stream);
    case 128:
        return rows <= 8 ? launch_nr<T, FMT, 128, 8>(a, rows, stream) : launch_nr<T, FMT, 128, 16>(a, rows, stream);
    default:  // 16 rows of 256 would not fit the registers
        return launch_nr<T, FMT, 256, 8>(a, rows, stream);
    }
}

template <typename T>
int launch_fmt(const TreeDev& a, int format, int D, int rows, cudaStream_t stream) {
    switch (format) {
    case QF_CACHE_PLAIN: return launch_d<T, QF_CACHE_PLAIN>(a, D, rows, stream);
    case QF_CACHE_E4M3: return launch_d<T, QF_CACHE_E4M3>(a, D, rows, stream);
    default: return launch_d<T, QF_CACHE_INT8>(a, D, rows, stream);
    }
}

}  // namespace

int launch_tree_mma(const TreeDev& a, int dtype, int format, int D, int rows, cudaStream_t stream) {
    return dtype == QF_F16 ? launch_fmt<__half>(a, format, D, rows, stream)
                           : launch_fmt<__nv_bfloat16>(a, format, D, rows, stream);
}

}  // namespace qf
