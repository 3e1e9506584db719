// Causal attention of runs of rows over a paged cache, on the matrix cores.
//
// A sequence's new rows and the kv_mul query heads of one KV head are packed
// into one list, head fastest: packed row x is row x / kv_mul, head x % kv_mul.
// All of them read the same K and V, so a tile of them is as good as a tile of
// rows of one head, whatever kv_mul is, and short runs fill a tile sooner.
//
// Tiling.  A workgroup has four waves: RG groups of 32 packed rows and KSP key
// splits (RG * KSP = 4).  A step stages KSP tiles of 32 keys in LDS, row by
// row and double-buffered: the next step's rows are on their way from their
// pages into registers while this one is attended, and the pages of the one
// after that are being looked up.  Keys are numbered without the window's gap
// (Visible of the workgroup's rows).  Per wave and tile, with 32x32 MFMAs:
//   S^T = K . Q^T    A = K rows, B = Q^T (registers): lane (n = l % 32, h = l /
//                    32) ends with the scores of packed row n against keys
//                    8 (r / 4) + 4 h + r % 4 in register r;
//   O^T = V^T . P^T  B = P^T: a lane supplies its own probabilities, so they
//                    never move between lanes; A = V^T with its keys in that
//                    order (bf16: a transposing LDS read; f32: plain reads).
//
// Precision.  f32 pages: v_mfma_f32_32x32x2_f32.  bf16 pages: K and V are bf16
// as they are; q and p are split into three bf16 values (24 bits, each the
// rounded remainder of the ones before), three v_mfma_f32_32x32x16_bf16 for a
// product, exact up to f32's rounding of the sums.  q is first scaled by a
// power of two per row, so that no value of any size leaves bf16's exponents;
// the scores' scale takes it back.
//
// What bounds it: the matrix cores for long runs (three bf16 products at 16
// times the f32 MFMA rate, or one f32 product), the softmax between them next.
#include <float.h>
#include <math.h>

#include "paged_common.h"
#include "slm_internal.h"

namespace slm {
namespace {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float v16 __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));
typedef unsigned int u2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int KT = 32;  // keys of a tile, packed rows of a wave

struct PrefillParams {
    PagedView b;
    const float* q;
    float* out;
    int num_heads;
    int kv_mul;
    int window;
    int sinks;
    float scale_log2;
};

// Distance of rows in LDS, in 16-byte chunks (16 of which are all banks).  A K
// read takes the same chunk of 32 rows: an odd distance gives 16 neighbouring
// rows all banks.  A V read takes four neighbouring chunks of rows 4 h + (0..3)
// (bf16, transposing: a distance of 4 or 12 modulo 16 spreads four rows over
// all banks) or eight of rows 4 h + r (f32: 2 modulo 4 puts the two rows side
// by side).  As the distances are constants, so are the offsets of a lane's
// reads; slots chosen by an exclusive or of row bits meet no conflicts either,
// but need an address register for each read.
constexpr int k_stride(int ch) { return ch | 1; }
constexpr int v_stride(bool bf, int ch) {
    if (!bf) return ch + (ch % 4 == 2 ? 0 : 2);
    while (ch % 16 != 4 && ch % 16 != 12) ch += 2;
    return ch;
}

// Two values as bf16 pairs: x = p1 + p2 + p3 (24 bits).
__device__ __forceinline__ void split2(float x0, float x1, uint32_t* p1, uint32_t* p2,
                                       uint32_t* p3) {
    const auto pack = [](float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, bf2));
    };
    *p1 = pack(x0, x1);
    x0 -= __uint_as_float(*p1 << 16);
    x1 -= __uint_as_float(*p1 & 0xFFFF0000u);
    *p2 = pack(x0, x1);
    x0 -= __uint_as_float(*p2 << 16);
    x1 -= __uint_as_float(*p2 & 0xFFFF0000u);
    *p3 = pack(x0, x1);
}

__device__ __forceinline__ void split8(const float* x, bf8 (&p)[3]) {
    u4 w[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t a, b, c;
        split2(x[2 * i], x[2 * i + 1], &a, &b, &c);
        w[0][i] = a, w[1][i] = b, w[2][i] = c;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) p[k] = __builtin_bit_cast(bf8, w[k]);
}

// The value of lane l ^ 32.
__device__ __forceinline__ float other_half(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float((threadIdx.x & 32) ? a[0] : a[1]);
}

template <class T>
__device__ __forceinline__ bool not_finite(u4 x) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2)
            any |= ((x[i] & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
        else
            any |= ((x[i] & 0x7F800000u) + 0x00800000u) & 0x80000000u;
    }
    return any != 0;
}

// A tile of packed rows of one sequence.
struct Tile {
    int seq;    // -1: none
    int index;  // within the sequence
    int row0;   // the sequence's first row of the batch
    int rows;   // and how many it has
};

// Tile `want` of the batch, the last one first (a sequence's last rows see the
// most keys).  Every lane of the wave gets the same answer.
template <int BM>
__device__ Tile find_tile(const PrefillParams& p, int want) {
    const PagedView& b = p.b;
    const int lane = threadIdx.x & 63;
    const auto rows_of = [&](int s, int* first) {
        const int lo = paged_min(paged_max(b.row_start[s], 0), b.n_rows);
        *first = lo;
        return paged_min(paged_max(b.row_start[s + 1], lo), b.n_rows) - lo;
    };
    const auto tiles_of = [&](int rows) {
        return (int)(((long long)rows * p.kv_mul + BM - 1) / BM);
    };
    int before = 0;
    for (int top = b.n_seqs; top > 0; top -= 64) {
        const int s = top - 1 - lane;  // lane 0 has the last sequence
        int first = 0, rows = 0, cnt = 0;
        if (s >= 0) {
            rows = rows_of(s, &first);
            cnt = tiles_of(rows);
        }
        int upto = cnt;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(upto, o);
            if (lane >= o) upto += y;
        }
        const unsigned long long m = __ballot(want < before + upto);
        if (m) {
            const int l = __ffsll(m) - 1;
            const int end = before + __builtin_amdgcn_readlane(upto, l);
            return Tile{__builtin_amdgcn_readfirstlane(top - 1 - l),
                        __builtin_amdgcn_readfirstlane(end - 1 - want),
                        __builtin_amdgcn_readlane(first, l), __builtin_amdgcn_readlane(rows, l)};
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return Tile{-1, 0, 0, 0};
}

template <class T, int HD, int KSP>
__global__ __launch_bounds__(kThreads, HD <= 128 ? 2 : 1) void paged_prefill_kernel(
    PrefillParams p) {
    constexpr bool BF = sizeof(T) == 2;
    constexpr int RG = 4 / KSP;            // groups of packed rows
    constexpr int BM = 32 * RG;            // packed rows of a workgroup
    constexpr int KS = KSP * KT;           // keys of a step
    constexpr int CV = 16 / sizeof(T);     // values of a chunk
    constexpr int CH = HD / CV;            // chunks of a row
    constexpr int NC = (KS * CH + kThreads - 1) / kThreads;  // a thread's chunks of K (and V)
    constexpr bool EXACT = KS * CH % kThreads == 0;
    constexpr int NQ = HD / 16;            // 16-dim steps of K . Q^T
    constexpr int ND = (HD + 31) / 32;     // 32-dim tiles of O^T
    constexpr bool DPAD = HD % 32 != 0;    // the last of them is half empty
    constexpr int KST = k_stride(CH), VST = v_stride(BF, CH);
    __shared__ u4 s_k[2][KS * KST], s_v[2][KS * VST];
    __shared__ float s_p[4][16][32];  // merge of the key splits; see `mixed` below
    __shared__ float s_ml[KSP > 1 ? 4 : 1][2][32];

    const PagedView& b = p.b;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, half = lane >> 5;
    const int rg = wave / KSP, ksp = wave % KSP;

    const int g = blockIdx.x % b.kv_heads;
    const Tile tile = find_tile<BM>(p, blockIdx.x / b.kv_heads);
    if (tile.seq < 0) return;  // uniform
    const int len = b.lens[tile.seq];
    const bool bad = len < 0 || len > b.max_len;
    const int packed = tile.rows * p.kv_mul;
    const int x0 = tile.index * BM;  // first packed row
    const int pos0 = bad ? -tile.rows : len - tile.rows;  // position of the sequence's first row
    const int x = x0 + rg * 32 + n;  // this lane's packed row
    const bool row_ok = x < packed;
    const int j = min(x, packed - 1) / p.kv_mul;
    const int head = g * p.kv_mul + min(x, packed - 1) - j * p.kv_mul;
    const int pos = pos0 + j;  // < 0: an empty row
    const int pos_out = p.window > 0 ? pos - p.window : -1;  // the last row behind the window
    // positions of the workgroup's first and last row
    const int pos_first = max(0, pos0 + x0 / p.kv_mul);
    const int pos_last = pos0 + (min(x0 + BM, packed) - 1) / p.kv_mul;
    // and of the wave's
    const int xw = x0 + rg * 32;
    const bool wave_ok = xw < packed;
    const int wpos_first = max(0, pos0 + xw / p.kv_mul);
    const int wpos_last = pos0 + (min(xw + 32, packed) - 1) / p.kv_mul;

    // the keys that any of the rows sees: Visible(pos_last), from the first
    // row's window on
    Visible vis(pos_last, 0, 0);
    if (pos_last >= 0 && p.window > 0) {
        vis.lo = max(0, pos_first + 1 - p.window);
        vis.first = min(p.sinks, vis.lo);
        vis.count = vis.first + pos_last + 1 - vis.lo;
    }
    const int steps = (vis.count + KS - 1) / KS;
    const T* pages = static_cast<const T*>(b.pages);
    const int32_t* table = b.table + (size_t)tile.seq * b.stride;
    const int slot_mask = (1 << b.ps_shift) - 1;
    const size_t to_v = ((size_t)b.kv_heads << b.ps_shift) * HD;

    // ---- staging ----
    int page[NC];
    u4 kr[NC], vr[NC];
    unsigned lost = 0;  // bit 2i: chunk i's page is bad; bit 2i + 1: it lies behind the end
    const auto key_of = [&](int st, int i) { return st * KS + (tid + i * kThreads) / CH; };
    const auto look_up = [&](int st) {
#pragma unroll
        for (int i = 0; i < NC; ++i)
            page[i] = table[vis.row(min(key_of(st, i), vis.count - 1)) >> b.ps_shift];
    };
    const auto fetch = [&](int st) {
        lost = 0;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int u = key_of(st, i);
            const bool ok = paged_page_ok(b, page[i]);
            if (!ok) lost |= 1u << (2 * i);
            if (u >= vis.count) lost |= 2u << (2 * i);
            const int t = vis.row(min(u, vis.count - 1));
            const T* at = pages + paged_at(b, ok ? page[i] : 0, 0, g, t & slot_mask, HD) +
                          (tid + i * kThreads) % CH * CV;
            kr[i] = *reinterpret_cast<const u4*>(at);
            vr[i] = *reinterpret_cast<const u4*>(at + to_v);
        }
    };
    // Into LDS.  Rows behind the end are zeros; of a bad page K is NaN, so that
    // the scores of the rows that see it are.  Whether V holds a value that is
    // not finite is asked for where some rows do not see it.
    const auto stage = [&](int buf, bool ask) {
        bool odd = false;
        if (__any(lost != 0)) {
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                if (lost & (3u << (2 * i))) {
                    const unsigned w = lost & (2u << (2 * i)) ? 0u : BF ? 0x7FC07FC0u : 0x7FC00000u;
                    kr[i] = u4{w, w, w, w};
                    vr[i] = u4{0, 0, 0, 0};
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int e = tid + i * kThreads, row = e / CH;
            if (!EXACT && row >= KS) break;
            s_k[buf][row * KST + e % CH] = kr[i];
            s_v[buf][row * VST + e % CH] = vr[i];
            if (ask) odd |= not_finite<T>(vr[i]);
        }
        return odd;
    };

    // ---- q ----
    // Lane (n, half) holds dims 16 i + 8 half + (0..7) of packed row n, times a
    // power of two for bf16 pages.
    float scale = p.scale_log2;
    bf8 qb[BF ? NQ : 1][3];
    float qf[BF ? 1 : NQ][8];
    {
        const float* src = p.q + ((size_t)(tile.row0 + j) * p.num_heads + head) * HD + 8 * half;
        float xq[NQ][8];
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const float4 a = ld4(src + 16 * i), c = ld4(src + 16 * i + 4);
            const float v[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) xq[i][e] = v[e];
        }
        if constexpr (BF) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < NQ; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(xq[i][e]));
            top = fmaxf(top, other_half(top));
            // largest magnitude in [2^-8, 2^-7): sums of hd products with any
            // bf16 K stay finite
            int ex = 0;
            if (top > 0.0f && top < INFINITY) {
                (void)frexpf(top, &ex);
                ex += 7;
            }
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
#pragma unroll
                for (int e = 0; e < 8; ++e) xq[i][e] = ldexpf(xq[i][e], -ex);
                split8(xq[i], qb[i]);
            }
            // (never 0: scores of -inf must stay -inf)
            scale = fmaxf(ldexpf(scale, ex), FLT_MIN);
        } else {
#pragma unroll
            for (int i = 0; i < NQ; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) qf[i][e] = xq[i][e];
        }
    }

    v16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = v16{};
    float m = -FLT_MAX, l = 0.0f;  // finite m: a row that has seen no key yet needs no guard

    // ---- one tile of the wave ----
    const auto attend = [&](int buf, int u0, bool mixed) {
        const u4* sk = &s_k[buf][ksp * KT * KST];
        const u4* sv = &s_v[buf][ksp * KT * VST];
        v16 s = v16{};
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            if constexpr (BF) {
                const bf8 kf = __builtin_bit_cast(bf8, sk[n * KST + 2 * i + half]);
#pragma unroll
                for (int k = 2; k >= 0; --k)
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qb[i][k], s, 0, 0, 0);
            } else {
                // dims 16 i + 8 half + (0..7), as q has them
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const u4 kf = sk[n * KST + 4 * i + 2 * half + c];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kf[e]),
                                                                 qf[i][4 * c + e], s, 0, 0, 0);
                }
            }
        }
        // Rows u0 .. u0 + 31 are t0 .. t0 + 31, or they lie on both sides of
        // the gap, or behind the end (then t > pos for every row).
        const int t0 = vis.row(u0);
        const bool gap = u0 < vis.first && u0 + KT > vis.first;
        const bool hidden = gap || t0 + KT - 1 > wpos_first ||
                            (p.window > 0 && u0 >= vis.first && t0 <= wpos_last - p.window);
        unsigned unseen = 0;
        if (hidden) {  // uniform
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int u = u0 + 8 * (r / 4) + 4 * half + r % 4;
                const int t = u + (u < vis.first ? 0 : vis.lo - vis.first);
                const bool hide = (t > pos) | ((t <= pos_out) & (t >= p.sinks));
                s[r] = hide ? -INFINITY : s[r];
                unseen |= (unsigned)hide << r;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        mx = fmaxf(mx, other_half(mx)) * scale;
        if (__any(mx > m + kLazyRescale)) {  // uniform
            const float mn = fmaxf(m, mx);
            const float alpha = fast_exp2(m - mn);
            l *= alpha;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= alpha;
            m = mn;
        }
        float ps = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = fast_exp2(fmaf(s[r], scale, -m));
            ps += s[r];
        }
        l += ps;
        if (mixed && hidden) {
            // V holds an infinity or a NaN, and some rows do not see some keys
            // (0 * inf is NaN in a product): one key after another, by the
            // rows that see it.
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    s_p[wave][8 * (r / 4) + 4 * half + r % 4][n] =
                        unseen >> (8 * ks + r) & 1 ? -1.0f : s[8 * ks + r];
                __builtin_amdgcn_wave_barrier();
                for (int k = 0; k < 16; ++k) {
                    const float pk = s_p[wave][k][n];
                    if (pk < 0.0f) continue;
                    const int row = 16 * ks + k;
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int dim = min(32 * d + 8 * (r / 4) + 4 * half + r % 4, HD - 1);
                            const T* c = reinterpret_cast<const T*>(
                                &sv[row * VST + dim / CV]);
                            o[d][r] = fmaf(pk, (float)c[dim % CV], o[d][r]);
                        }
                }
                __builtin_amdgcn_wave_barrier();
            }
            return;
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if constexpr (BF) {
                bf8 pf[3];
                const float xs[8] = {s[8 * ks],     s[8 * ks + 1], s[8 * ks + 2], s[8 * ks + 3],
                                     s[8 * ks + 4], s[8 * ks + 5], s[8 * ks + 6], s[8 * ks + 7]};
                split8(xs, pf);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    // 16 lanes read a 4 x 16 block row by row and get it column
                    // by column; dims behind HD repeat others
                    const int dim = DPAD && d == ND - 1 ? 4 * (lane & 3)
                                                        : 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                    s4 w[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int row = 16 * ks + 8 * c + 4 * half + ((lane >> 2) & 3);
                        const T* at = reinterpret_cast<const T*>(&sv[row * VST]) + 32 * d + dim;
                        w[c] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s4*)(at));
                    }
                    const u2 w0 = __builtin_bit_cast(u2, w[0]), w1 = __builtin_bit_cast(u2, w[1]);
                    const bf8 vf = __builtin_bit_cast(bf8, u4{w0[0], w0[1], w1[0], w1[1]});
#pragma unroll
                    for (int k = 2; k >= 0; --k)
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[k], o[d], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const int dim = 32 * d + (DPAD && d == ND - 1 ? n & 15 : n);
#pragma unroll
                    for (int r = 8 * ks; r < 8 * ks + 8; ++r) {
                        const int row = 8 * (r / 4) + 4 * half + r % 4;
                        const float v = reinterpret_cast<const float*>(&sv[row * VST])[dim];
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[r], o[d], 0, 0, 0);
                    }
                }
            }
        }
    };

    // ---- the steps ----
    if (steps > 0) {  // uniform
        look_up(0);
        fetch(0);
        if (steps > 1) look_up(1);
        for (int st = 0; st < steps; ++st) {
            const int u = st * KS, t = vis.row(u);
            // some row of the workgroup does not see some key of the step
            const bool ask = u + KS > vis.count || t + KS - 1 > pos_first || p.window > 0;
            const bool odd = stage(st & 1, ask);
            if (st + 1 < steps) {
                fetch(st + 1);
                if (st + 2 < steps) look_up(st + 2);
            }
            bool mixed = false;
            if (ask)
                mixed = __syncthreads_or(odd);
            else
                __syncthreads();
            const int u0 = u + ksp * KT;
            // a wave whose rows are all empty or in front of the tile has
            // nothing to do there
            if (wave_ok && u0 < vis.count && vis.row(u0) <= wpos_last) attend(st & 1, u0, mixed);
        }
    }
    l += other_half(l);

    // ---- key splits, then the output ----
    if constexpr (KSP > 1) {
        // every wave scales its state to the row's max over the splits, split 0
        // adds the others' in order
        if (half == 0) {
            s_ml[wave][0][n] = m;
            s_ml[wave][1][n] = l;
        }
        __syncthreads();
        float top = m;
#pragma unroll
        for (int k = 0; k < KSP; ++k) top = fmaxf(top, s_ml[rg * KSP + k][0][n]);
        const float e = fast_exp2(m - top);
        l = 0.0f;
#pragma unroll
        for (int k = 0; k < KSP; ++k)
            l += s_ml[rg * KSP + k][1][n] * fast_exp2(s_ml[rg * KSP + k][0][n] - top);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            o[d] *= e;
            if (ksp)
#pragma unroll
                for (int r = 0; r < 16; ++r) s_p[wave][2 * r + half][n] = o[d][r];
            __syncthreads();
            if (!ksp)
#pragma unroll
                for (int k = 1; k < KSP; ++k)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] += s_p[wave + k][2 * r + half][n];
            __syncthreads();
        }
        if (ksp) return;
    }
    if (!row_ok) return;
    // an empty row gives zeros, one of a bad length NaN
    const float inv = bad ? __builtin_nanf("") : pos < 0 ? 0.0f : 1.0f / l;
    float* dst = p.out + ((size_t)(tile.row0 + j) * p.num_heads + head) * HD;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int dim = 32 * d + 8 * (r / 4) + 4 * half;
            if (DPAD && d == ND - 1 && r >= 8) break;
            *reinterpret_cast<float4*>(dst + dim) = make_float4(o[d][r] * inv, o[d][r + 1] * inv,
                                                                o[d][r + 2] * inv, o[d][r + 3] * inv);
        }
}

template <class T, int HD, int KSP>
hipError_t launch_k(const Shape& s, const PrefillParams& p, hipStream_t st) {
    constexpr int BM = 32 * (4 / KSP);
    // at most this many tiles, whatever the rows' division among the sequences
    const long tiles = (long)p.b.n_rows * s.kv_mul / BM + p.b.n_seqs;
    const long wgs = tiles * s.num_kv_heads;
    if (wgs >= (1L << 32) / kThreads) return hipErrorInvalidValue;
    hipLaunchKernelGGL((paged_prefill_kernel<T, HD, KSP>), dim3((unsigned)wgs), dim3(kThreads), 0,
                       st, p);
    return hipGetLastError();
}

template <class T, int HD>
hipError_t launch_t(const Shape& s, const PrefillParams& p, hipStream_t st) {
    return launch_k<T, HD, 1>(s, p, st);
}

template <class T>
hipError_t launch_hd(const Shape& s, const PrefillParams& p, hipStream_t st) {
    switch (s.head_dim) {
        case 16: return launch_t<T, 16>(s, p, st);
        case 32: return launch_t<T, 32>(s, p, st);
        case 48: return launch_t<T, 48>(s, p, st);
        case 64: return launch_t<T, 64>(s, p, st);
        case 96: return launch_t<T, 96>(s, p, st);
        case 128: return launch_t<T, 128>(s, p, st);
        case 256: return launch_t<T, 256>(s, p, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_paged_prefill(const Shape& s, const PagedView& b, bool bf16, const float* q,
                                int window, int sinks, float* out, hipStream_t st) {
    const PrefillParams p{b,      q,     out, s.num_heads, s.kv_mul, window,
                          sinks, 1.4426950408889634f / sqrtf((float)s.head_dim)};
    return bf16 ? launch_hd<__bf16>(s, p, st) : launch_hd<float>(s, p, st);
}

}  // namespace slm
