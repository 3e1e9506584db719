// Attention of single rows over a paged cache: each row's keys are cut into
// chunks, a workgroup attends one chunk with the query heads of one KV head,
// and a second kernel joins the chunks.
//
//   out_h = sum_t softmax_t(q_h . K[t, g] / sqrt(hd)) V[t, g]   over the rows
//   t that the row sees, g = h / kv_mul
//
// What bounds it: the K and V rows, read once each for up to four query heads
// of the KV head.  The softmax is one pass (running max m and sum l, log2
// domain), so nothing else of that size moves.  Measured, Llama-3-8B shape: 8 rows
// with a window of 4096, f32 (238 MB) 38.6 us back to back, 6.2 TB/s; 32 rows of up
// to 4223 keys, bf16 (300 MB) 56 us, 5.3 TB/s; one row of 32768, bf16 (134 MB) 22.8
// us, 5.9 TB/s.  A streaming read reaches 6.9.
//
// Chunks.  A batch's sequences differ in length, and the host does not know
// the lengths (they lie on the device, so that a captured graph follows them).
// Every wave therefore forms the same plan from them: with T_r the tiles of
// row r's visible keys (one at least), T their sum and U the workgroups per KV
// head group that fill the card, a chunk is C = ceil(T / U) tiles and row r has
// ceil(T_r / C) chunks, at most U + n_rows together, which is the grid;
// workgroups behind the last chunk end at once.  Where C would exceed
// kLongChunk tiles, more and shorter chunks even out the CUs' loads: up to 4 U, of kChunk
// tiles at least (64 sequences of up to 4201 rows, Llama-3-8B shape in bf16: 118
// us with U, 99 us with 4 U; 16 of them 35.7 and 38.8).  A row of one chunk is
// written to out directly.
//
// Lanes.  LPG lanes hold one key's head_dim values in 16-byte loads, so a wave
// attends 64 / LPG keys at a time, each lane group with its own (m, l, o); the
// states are merged through LDS at the end.  Keys are numbered without the
// window's gap (Visible), and each lane group looks its page up a tile ahead.
// With four query heads to a bf16 key the vector unit would be the bound: their
// scores come from the matrix cores (matrix_scores), from q split into three
// bf16 planes, which K needs not be.
#include <float.h>
#include <math.h>

#include <algorithm>

#include "paged_common.h"
#include "slm_internal.h"

namespace slm {
namespace {

typedef float v4 __attribute__((ext_vector_type(4)));

// 16 bytes of the cache as floats
template <class T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(u4 x, float (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(x[i]);
    }
};
template <>
struct Vec<__bf16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(u4 x, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(x[i] << 16);
            f[2 * i + 1] = __uint_as_float(x[i] & 0xFFFF0000u);
        }
    }
};

// Lanes per key (LPG) and keys per lane group and tile (TP).
template <class T, int HD>
struct Cfg;
template <> struct Cfg<float, 16> { static constexpr int LPG = 2, TP = 2; };
template <> struct Cfg<float, 32> { static constexpr int LPG = 4, TP = 2; };
template <> struct Cfg<float, 48> { static constexpr int LPG = 4, TP = 2; };
template <> struct Cfg<float, 64> { static constexpr int LPG = 8, TP = 2; };
template <> struct Cfg<float, 96> { static constexpr int LPG = 8, TP = 2; };
template <> struct Cfg<float, 128> { static constexpr int LPG = 16, TP = 2; };
template <> struct Cfg<float, 256> { static constexpr int LPG = 32, TP = 2; };
template <> struct Cfg<__bf16, 16> { static constexpr int LPG = 2, TP = 2; };
template <> struct Cfg<__bf16, 32> { static constexpr int LPG = 4, TP = 2; };
template <> struct Cfg<__bf16, 48> { static constexpr int LPG = 2, TP = 1; };
template <> struct Cfg<__bf16, 64> { static constexpr int LPG = 8, TP = 4; };
template <> struct Cfg<__bf16, 96> { static constexpr int LPG = 4, TP = 1; };
template <> struct Cfg<__bf16, 128> { static constexpr int LPG = 16, TP = 4; };
template <> struct Cfg<__bf16, 256> { static constexpr int LPG = 32, TP = 4; };

constexpr int kWaves = 4;
constexpr int kXcds = 8;
constexpr int kMaxGb = 4;  // query heads of a workgroup, at most
// Tiles up to which no row is split: a tile costs its workgroup about 1 us, the
// second launch that joins chunks 4.
constexpr int kWholeTiles = 4;

template <class T, int HD>
constexpr int tile_rows() {
    return kWaves * (64 / Cfg<T, HD>::LPG) * Cfg<T, HD>::TP;
}

struct DecodeParams {
    PagedView b;
    const float* q;   // [n_rows][dim], rotated
    float* out;       // [n_rows][dim]
    float* part_o;    // [chunk][num_heads][head_dim]
    float* part_ml;   // [chunk][num_heads][2]
    int units;        // U, chunks to aim for; 0: every row is one chunk
    int most_units;   // and where they would exceed kChunk tiles
    int num_heads;
    int kv_mul;
    int gb;           // query heads of a workgroup
    int window;
    int sinks;
    float scale_log2;
};

// Where chunk `want` of the batch (or the first chunk of row `row_want`) lies.
constexpr int kChunk = 8, kLongChunk = 16;

__device__ __forceinline__ int chunk_tiles(const DecodeParams& p, int total) {  // (0 < total < 2^30)
    const int c = (total + p.units - 1) / p.units;
    return c <= kLongChunk ? c : max(kChunk, (total + p.most_units - 1) / p.most_units);
}

struct Chunk {
    int row;     // -1: behind the last chunk
    int index;   // within its row
    int count;   // of its row
    int tiles;   // C
    int first;   // the row's first chunk
};

template <int TILE>
__device__ __forceinline__ int row_tiles(const DecodeParams& p, int row) {
    const PagedRow r = paged_row(p.b, row);
    return max(1, (Visible(r.pos, p.window, p.sinks).count + TILE - 1) / TILE);
}

// Every lane of the wave gets the same answer.
template <int TILE>
__device__ Chunk find_chunk(const DecodeParams& p, int want, int row_want) {
    const int n = p.b.n_rows;
    if (n == 1) {  // nothing to look for
        const int t = row_tiles<TILE>(p, 0), c = chunk_tiles(p, t);
        const int k = (t + c - 1) / c;
        return Chunk{want < k ? 0 : -1, want, k, c, 0};
    }
    const int lane = threadIdx.x & 63;
    const int mine0 = lane < n ? row_tiles<TILE>(p, lane) : 0;
    int total = mine0;
    for (int r = lane + 64; r < n; r += 64) total += row_tiles<TILE>(p, r);
    const int c = __builtin_amdgcn_readfirstlane(chunk_tiles(p, wave_total(total)));
    int before = 0;  // chunks of the rows in front of this stretch of 64
    for (int r0 = 0; r0 < n; r0 += 64) {
        const int mine = !r0 ? mine0 : r0 + lane < n ? row_tiles<TILE>(p, r0 + lane) : 0;
        const int cnt = (mine + c - 1) / c;
        const int upto = wave_upto(cnt);  // chunks up to this lane's row
        const bool here = row_want >= 0 ? r0 + lane == row_want
                                        : lane + r0 < n && want < before + upto;
        const unsigned long long m = __ballot(here);
        if (m) {
            const int l = __ffsll(m) - 1;
            const int k = __builtin_amdgcn_readlane(cnt, l);
            const int first = before + __builtin_amdgcn_readlane(upto, l) - k;
            return Chunk{__builtin_amdgcn_readfirstlane(r0 + l),
                         __builtin_amdgcn_readfirstlane(want - first), k, c,
                         __builtin_amdgcn_readfirstlane(first)};
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return Chunk{-1, 0, 0, c, 0};
}

// One online-softmax step over TP keys of a lane group (the first `TP` of the
// raw registers): the state is rescaled only when some lane's max has grown by
// more than kLazyRescale.
template <class T, int HD, int LPG, int NV, int GB, int TP, int TPR>
__device__ __forceinline__ void attend(const float (&q)[GB][NV][Vec<T>::N], const u4 (&kr)[TPR][NV],
                                       const u4 (&vr)[TPR][NV], int at, float (&m)[GB],
                                       float (&l)[GB], float (&o)[GB][NV][Vec<T>::N]) {
    constexpr int N = Vec<T>::N;
    float sc[GB][TP];
#pragma unroll
    for (int t = 0; t < TP; ++t) {
#pragma unroll
        for (int i = 0; i < GB; ++i) sc[i][t] = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float f[N];
            Vec<T>::get(kr[at + t][v], f);
#pragma unroll
            for (int i = 0; i < GB; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) sc[i][t] = fmaf(q[i][v][e], f[e], sc[i][t]);
        }
    }
    float pr[GB][TP];
#pragma unroll
    for (int i = 0; i < GB; ++i) {
#pragma unroll
        for (int t = 0; t < TP; ++t) sc[i][t] = group_sum<LPG>(sc[i][t]);
        float mx = sc[i][0];
#pragma unroll
        for (int t = 1; t < TP; ++t) mx = fmaxf(mx, sc[i][t]);
        if (__any(mx > m[i] + kLazyRescale)) {  // uniform
            const float mn = fmaxf(m[i], mx);
            const float alpha = fast_exp2(m[i] - mn);
            l[i] *= alpha;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < N; ++e) o[i][v][e] *= alpha;
            m[i] = mn;
        }
#pragma unroll
        for (int t = 0; t < TP; ++t) {
            pr[i][t] = fast_exp2(sc[i][t] - m[i]);
            l[i] += pr[i][t];
        }
    }
#pragma unroll
    for (int t = 0; t < TP; ++t)
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float f[N];
            Vec<T>::get(vr[at + t][v], f);
#pragma unroll
            for (int i = 0; i < GB; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) o[i][v][e] = fmaf(pr[i][t], f[e], o[i][v][e]);
        }
}

// Scores by the matrix cores: for four heads of whole 32-dim steps whose V rows
// fill no more than 16 lanes; of hd 96, where a lane holds 24 dims and three
// heads already leave two waves to a SIMD, also for three.  64 sequences of up
// to 4201 bf16 rows, 8 KV heads (hd 96 and three heads: 4), against the vector
// unit (us): 4 heads of 128 98 / 108, of 96 59 / 112, of 64 59 / 66, of 32 37 /
// 40; 3 heads of 128 57 / 55, of 96 55 / 92, of 64 31 / 28.
template <class T, int HD, int GB>
constexpr bool matrix_scores() {
    return sizeof(T) == 2 && HD % 32 == 0 && HD <= 128 && (GB == 4 || (GB == 3 && HD == 96));
}

// x of lane i of the quad
template <int I>
__device__ __forceinline__ float quad_lane(float x) {
    return __uint_as_float(
        __builtin_amdgcn_mov_dpp(__float_as_uint(x), I * 0x55, 0xF, 0xF, true));
}
__device__ __forceinline__ float quad_lane(float x, int i) {  // i: a constant where it is used
    return i == 0 ? quad_lane<0>(x) : i == 1 ? quad_lane<1>(x) : i == 2 ? quad_lane<2>(x)
                                                                       : quad_lane<3>(x);
}

// REUSE: another workgroup reads the same keys for other heads.
template <class T, int HD, int GB, bool REUSE>
__global__ __launch_bounds__(64 * kWaves) void paged_decode_kernel(DecodeParams p) {
    constexpr bool MX = matrix_scores<T, HD, GB>();
    constexpr int LPG = Cfg<T, HD>::LPG, TP = Cfg<T, HD>::TP, N = Vec<T>::N;
    constexpr int NV = HD / LPG / N;
    constexpr int GPW = 64 / LPG;
    constexpr int TILE = tile_rows<T, HD>();
    constexpr int NS = kWaves * GPW;  // lane-group states of the workgroup
    static_assert(HD % (LPG * N) == 0, "whole 16-byte loads");
    const PagedView& b = p.b;

    // Workgroups go to the XCDs round-robin: the nhb that read the same keys for
    // different heads are kXcds apart, so that one L2 serves them all, by plain
    // loads (16 sequences of up to 4201 rows, 8 heads to the KV head at hd 128: f32
    // 32.2 us side by side, 23.3 apart, 25.1 with nontemporal loads; bf16 22.1,
    // 18.2, 21.0).  Keys read once keep nontemporal loads (64 sequences, 4 heads:
    // f32 182 us against 202, bf16 99 against 109).
    const int nhb = (p.kv_mul + GB - 1) / GB;
    const int eight = blockIdx.x / kXcds;
    const int pair = eight / nhb * kXcds + blockIdx.x % kXcds;  // of a chunk and a KV head
    const int idx = pair / b.kv_heads;
    const int g = pair - idx * b.kv_heads;
    const int hb = eight % nhb * GB;  // this workgroup's heads in the KV head's kv_mul
    const int h0 = g * p.kv_mul + hb;

    Chunk ch{idx, 0, 1, 0, 0};
    if (!p.units) {
        if (idx >= b.n_rows) return;
    } else {
        ch = find_chunk<TILE>(p, idx, -1);
        if (ch.row < 0) return;
    }
    const PagedRow r = paged_row(b, ch.row);
    if (r.seq < 0) return;
    const Visible vis(r.pos, p.window, p.sinks);
    const int u_beg = ch.index * ch.tiles * TILE;
    const int u_end = ch.count == 1 ? vis.count : min(vis.count, u_beg + ch.tiles * TILE);

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane % LPG;
    const int lg = lane / LPG;
    const T* pages = static_cast<const T*>(b.pages);
    const int32_t* table = b.table + (size_t)r.seq * b.stride;
    const int slot_mask = (1 << b.ps_shift) - 1;

    float m[GB], l[GB], o[GB][NV][N];
#pragma unroll
    for (int i = 0; i < GB; ++i) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < N; ++e) o[i][v][e] = 0.0f;
        m[i] = -FLT_MAX;  // finite, so that m - m and score - m need no guard
        l[i] = 0.0f;
    }
    bool bad_page = false;
    const size_t to_v = ((size_t)b.kv_heads << b.ps_shift) * HD;
    const auto load = [](const T* a) {
        return REUSE ? *reinterpret_cast<const u4*>(a)
                     : __builtin_nontemporal_load(reinterpret_cast<const u4*>(a));
    };
    const auto q_row = [&](int i) {
        // a head group's last workgroup may have fewer heads: it computes one twice
        return p.q + ((size_t)ch.row * p.num_heads + g * p.kv_mul + min(hb + i, p.kv_mul - 1)) * HD;
    };
    if constexpr (MX) {
        // A wave has 16 DT keys of a tile.  S^T = K . Q^T by
        // v_mfma_f32_16x16x32_bf16: A is K as it lies in the page (lane l has
        // 16-byte pieces of key l % 16); the columns of B are the heads' three
        // bf16 planes, column 4 p + i plane p of head i.  Lane l ends with the
        // scores of head l % 4 against keys 4 (l / 16) + r, and the lane groups of
        // its row of 16 lanes take just these keys' V.  For four heads of 128 that
        // leaves 14 vector instructions per key of 29.
        constexpr int DT = TP * GPW / 16, NK = HD / 32, B = 16 / LPG, R = 4 / B;
        static_assert(TP == DT * R, "a row of 16 lanes takes the V of its four keys");
        const int row16 = lane >> 4, n = lane & 15, sub = n / LPG;
        bf8 qf[NK];
        float scale;
        {
            const float* src = q_row(min(n & 3, GB - 1));
            float x[NK][8], top = 0.0f;
#pragma unroll
            for (int i = 0; i < NK; ++i)
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const float4 y = ld4(src + 8 * (4 * i + row16) + e);
                    x[i][e] = y.x * p.scale_log2;
                    x[i][e + 1] = y.y * p.scale_log2;
                    x[i][e + 2] = y.z * p.scale_log2;
                    x[i][e + 3] = y.w * p.scale_log2;
                }
#pragma unroll
            for (int i = 0; i < NK; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][e]));
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            // largest magnitude in [2^-10, 2^-9), as for runs of rows
            int ex = 0;
            if (top > 0.0f && top < INFINITY) {
                (void)frexpf(top, &ex);
                ex += 9;
            }
            scale = ldexpf(1.0f, min(max(ex, -126), 127));
#pragma unroll
            for (int i = 0; i < NK; ++i) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][e] = ldexpf(x[i][e], -ex);
                bf8 w[3];
                split8(x[i], w);
                const u4 zero = {0, 0, 0, 0};
                qf[i] = n < 4 ? w[0] : n < 8 ? w[1] : n < 12 ? w[2]
                                                             : __builtin_bit_cast(bf8, zero);
            }
        }
        float mh = -FLT_MAX, lh = 0.0f;  // of head lane % 4 and this row of lanes' keys
        int page[DT];
        const auto key = [&](int tb, int t, int k) {
            return vis.row(min(tb + (wave * DT + t) * 16 + k, u_end - 1));
        };
        const auto look_up = [&](int tb) {
#pragma unroll
            for (int t = 0; t < DT; ++t) page[t] = table[key(tb, t, n) >> b.ps_shift];
        };
        if (u_beg < u_end) look_up(u_beg);
        for (int tb = u_beg; tb < u_end; tb += TILE) {
            u4 kr[DT][NK], vr[TP][NV];
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const bool ok = paged_page_ok(b, page[t]);
                bad_page |= !ok;
                const size_t off =
                    paged_at(b, ok ? page[t] : 0, 0, g, key(tb, t, n) & slot_mask, HD);
#pragma unroll
                for (int i = 0; i < NK; ++i) kr[t][i] = load(pages + off + 8 * (4 * i + row16));
#pragma unroll
                for (int s = 0; s < R; ++s) {  // lane k of a row has key k's address
                    const int k = 4 * row16 + sub * R + s;
                    const size_t voff = (size_t)(uint32_t)__shfl((int)(off >> 32), k) << 32 |
                                        (uint32_t)__shfl((int)off, k);
#pragma unroll
                    for (int v = 0; v < NV; ++v)
                        vr[t * R + s][v] = load(pages + to_v + voff + N * (v * LPG + li));
                }
            }
            if (tb + TILE < u_end) look_up(tb + TILE);
            v4 sc[DT];
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                v4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < NK; ++i)
                    s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, kr[t][i]),
                                                                qf[i], s, 0, 0, 0);
                // the planes' sum, the same bits in all four lanes of a head
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[r] += __uint_as_float(__builtin_amdgcn_mov_dpp(
                        __float_as_uint(s[r]), 0x128, 0xF, 0xF, true));  // row_ror:8
                    s[r] += __uint_as_float(__builtin_amdgcn_mov_dpp(
                        __float_as_uint(s[r]), 0x124, 0xF, 0xF, true));  // row_ror:4
                }
                sc[t] = s * scale;
            }
            if (tb + TILE > u_end) {  // uniform: the last keys; what lies behind has no part
                const int end = u_end - tb - wave * DT * 16;
#pragma unroll
                for (int t = 0; t < DT; ++t) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        sc[t][r] = 16 * t + 4 * row16 + r < end ? sc[t][r] : -INFINITY;
#pragma unroll
                    for (int s = 0; s < R; ++s)
#pragma unroll
                        for (int v = 0; v < NV; ++v) {
                            const bool in = 16 * t + 4 * row16 + sub * R + s < end;
                            const u4 zero = {0, 0, 0, 0};
                            vr[t * R + s][v] = in ? vr[t * R + s][v] : zero;
                        }
                }
            }
            float mx = sc[0][0];
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[t][r]);
            if (__any(mx > mh + kLazyRescale)) {  // uniform
                const float mn = fmaxf(mh, mx);
                const float alpha = fast_exp2(mh - mn);
                lh *= alpha;
                mh = mn;
#pragma unroll
                for (int i = 0; i < GB; ++i) {
                    const float a = quad_lane(alpha, i);
#pragma unroll
                    for (int v = 0; v < NV; ++v)
#pragma unroll
                        for (int e = 0; e < N; ++e) o[i][v][e] *= a;
                }
            }
#pragma unroll
            for (int t = 0; t < DT; ++t) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    sc[t][r] = fast_exp2(sc[t][r] - mh);
                    lh += sc[t][r];
                }
#pragma unroll
                for (int s = 0; s < R; ++s) {
                    float pr = sc[t][s];
#pragma unroll
                    for (int k = 1; k < B; ++k) pr = sub == k ? sc[t][k * R + s] : pr;
                    float pi[GB];
#pragma unroll
                    for (int i = 0; i < GB; ++i) pi[i] = quad_lane(pr, i);
#pragma unroll
                    for (int v = 0; v < NV; ++v) {
                        float f[N];
                        Vec<T>::get(vr[t * R + s][v], f);
#pragma unroll
                        for (int i = 0; i < GB; ++i)
#pragma unroll
                            for (int e = 0; e < N; ++e)
                                o[i][v][e] = fmaf(pi[i], f[e], o[i][v][e]);
                    }
                }
            }
        }
        bad_page = __any(bad_page);
#pragma unroll
        for (int i = 0; i < GB; ++i) {
            m[i] = quad_lane(mh, i);
            l[i] = sub == 0 ? quad_lane(lh, i) : 0.0f;  // once for a row of lanes
        }
    } else {
        float q[GB][NV][N];
#pragma unroll
        for (int i = 0; i < GB; ++i) {
            const float* src = q_row(i);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < N; e += 4) {
                    const float4 x = ld4(src + N * (v * LPG + li) + e);
                    q[i][v][e] = x.x * p.scale_log2;
                    q[i][v][e + 1] = x.y * p.scale_log2;
                    q[i][v][e + 2] = x.z * p.scale_log2;
                    q[i][v][e + 3] = x.w * p.scale_log2;
                }
        }

        int page[TP];
        const auto key = [&](int tb, int tp) {  // the lane group's key of a tile, clamped to the last
            return vis.row(min(tb + (tp * kWaves + wave) * GPW + lg, u_end - 1));
        };
        const auto look_up = [&](int tb) {
#pragma unroll
            for (int tp = 0; tp < TP; ++tp) page[tp] = table[key(tb, tp) >> b.ps_shift];
        };
        if (u_beg < u_end) look_up(u_beg);
        for (int tb = u_beg; tb < u_end; tb += TILE) {
            u4 kr[TP][NV], vr[TP][NV];
#pragma unroll
            for (int tp = 0; tp < TP; ++tp) {
                const bool ok = paged_page_ok(b, page[tp]);
                bad_page |= !ok;
                const T* at = pages + paged_at(b, ok ? page[tp] : 0, 0, g, key(tb, tp) & slot_mask, HD);
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    const T* a = at + N * (v * LPG + li);
                    kr[tp][v] = load(a);
                    vr[tp][v] = load(a + to_v);
                }
            }
            if (tb + TILE < u_end) look_up(tb + TILE);
            if (tb + TILE <= u_end) {
                attend<T, HD, LPG, NV, GB, TP, TP>(q, kr, vr, 0, m, l, o);
            } else {
                // the last keys: lane groups behind the end sit out, so that what
                // they loaded is never multiplied
#pragma unroll
                for (int tp = 0; tp < TP; ++tp)
                    if (tb + (tp * kWaves + wave) * GPW + lg < u_end)
                        attend<T, HD, LPG, NV, GB, 1, TP>(q, kr, vr, tp, m, l, o);
            }
        }
    }

    // Merge: every lane group scales its state to the workgroup's max into a
    // slot of its own, each thread sums the slots of one (head, dim).  As many
    // heads at a time as fit 40 KiB, so that the slots do not limit the
    // workgroups of a CU.
    constexpr int HR = NS * GB * HD * 4 <= 40 * 1024 ? GB : 1;
    __shared__ float s_m[kWaves][GB];
    __shared__ __align__(16) float s_o[NS][HR][HD];
    __shared__ float s_l[GB][NS];
    const float nan = __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < GB; ++i) {
        const float x = groups_max<LPG>(m[i]);
        if (lane == 0) s_m[wave][i] = x;
    }
    __syncthreads();
    const int slot = wave * GPW + lg;
#pragma unroll
    for (int i0 = 0; i0 < GB; i0 += HR) {
        if (i0) __syncthreads();
#pragma unroll
        for (int j = 0; j < HR; ++j) {
            const int i = i0 + j;
            float mw = s_m[0][i];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) mw = fmaxf(mw, s_m[w][i]);
            const float e = fast_exp2(m[i] - mw);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int k = 0; k < N; k += 4)
                    *reinterpret_cast<float4*>(&s_o[slot][j][N * (v * LPG + li) + k]) =
                        make_float4(o[i][v][k] * e, o[i][v][k + 1] * e, o[i][v][k + 2] * e,
                                    o[i][v][k + 3] * e);
            if (li == 0) s_l[i][slot] = bad_page ? nan : l[i] * e;
        }
        __syncthreads();
        for (int x = threadIdx.x; x < HR * HD; x += 64 * kWaves) {
            const int j = x / HD, d = x - j * HD, i = i0 + j;
            if (hb + i >= p.kv_mul) break;
            float so = 0.0f, sl = 0.0f;
            for (int s = 0; s < NS; ++s) {
                so += s_o[s][j][d];
                sl += s_l[i][s];
            }
            const int h = h0 + i;
            if (ch.count == 1) {
                // an empty row gives zeros, one of a bad length NaN
                p.out[((size_t)ch.row * p.num_heads + h) * HD + d] =
                    r.bad ? nan : vis.count ? so / sl : 0.0f;
            } else {
                const size_t at = (size_t)idx * p.num_heads + h;
                p.part_o[at * HD + d] = so;
                if (d == 0) {
                    float mw = s_m[0][i];
#pragma unroll
                    for (int w = 1; w < kWaves; ++w) mw = fmaxf(mw, s_m[w][i]);
                    p.part_ml[2 * at] = mw;
                    p.part_ml[2 * at + 1] = sl;
                }
            }
        }
    }
}

// Joins a row's chunks for one head: a workgroup per (row, head).  Lane groups of
// HD / 4 lanes go through every R-th chunk each, four at a time in flight, with a
// running max; their states are added through LDS in order.  Bound by its launch
// and two round trips to memory: 4.1 to 5 us.
template <class T, int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(DecodeParams p) {
    constexpr int TILE = tile_rows<T, HD>();
    constexpr int L4 = HD / 4, R = 256 / L4, B = 4;
    __shared__ float s_m[R], s_l[R];
    __shared__ __align__(16) float s_o[R][HD];
    const int row = blockIdx.x / p.num_heads;
    const int h = blockIdx.x - row * p.num_heads;
    const Chunk ch = find_chunk<TILE>(p, 0, row);
    if (ch.count == 1) return;  // written by its workgroup
    const int t = threadIdx.x;
    const int k = t / L4, d = t - k * L4;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
    if (k < R) {
        float m = -FLT_MAX, l = 0.0f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c0 = k; c0 < ch.count; c0 += B * R) {
            float2 y[B];
            float4 z[B];
#pragma unroll
            for (int i = 0; i < B; ++i) {  // behind the last chunk: the last once more
                const size_t at =
                    (size_t)(ch.first + min(c0 + i * R, ch.count - 1)) * p.num_heads + h;
                y[i] = ml[at];
                z[i] = ld4(p.part_o + at * HD + 4 * d);
            }
            float mn = m;
#pragma unroll
            for (int i = 0; i < B; ++i) mn = fmaxf(mn, y[i].x);
            const float a = fast_exp2(m - mn);
            m = mn;
            l *= a;
            o.x *= a, o.y *= a, o.z *= a, o.w *= a;
#pragma unroll
            for (int i = 0; i < B; ++i) {
                if (c0 + i * R >= ch.count) break;
                const float e = fast_exp2(y[i].x - m);
                l = fmaf(e, y[i].y, l);
                o.x = fmaf(e, z[i].x, o.x);
                o.y = fmaf(e, z[i].y, o.y);
                o.z = fmaf(e, z[i].z, o.z);
                o.w = fmaf(e, z[i].w, o.w);
            }
        }
        if (d == 0) {
            s_m[k] = m;
            s_l[k] = l;
        }
        *reinterpret_cast<float4*>(&s_o[k][4 * d]) = o;
    }
    __syncthreads();
    if (t < HD) {
        const int n = min(R, ch.count);
        float mx = s_m[0], so = 0.0f, sl = 0.0f;
        for (int i = 1; i < n; ++i) mx = fmaxf(mx, s_m[i]);
        for (int i = 0; i < n; ++i) {
            const float e = fast_exp2(s_m[i] - mx);
            sl = fmaf(e, s_l[i], sl);
            so = fmaf(e, s_o[i][t], so);
        }
        p.out[((size_t)row * p.num_heads + h) * HD + t] = so / sl;
    }
}

// Query heads of a workgroup: kv_mul in equal parts of at most four (eight took
// 1.3 to 2 times as long: half the waves fit).
int gb_of(int kv_mul) {
    const int parts = (kv_mul + kMaxGb - 1) / kMaxGb;
    return (kv_mul + parts - 1) / parts;
}

// Workgroups per KV head group that fill the card with two waves per SIMD.
int units_of(const Shape& s, int groups) {
    const int wgs = 2 * s.cus;
    return groups >= wgs ? 1 : wgs / groups;
}

int groups_of(const Shape& s) {
    const int gb = gb_of(s.kv_mul);
    return s.num_kv_heads * ((s.kv_mul + gb - 1) / gb);
}

template <class T, int HD>
hipError_t launch_t(const Shape& s, DecodeParams p, hipStream_t st) {
    const int groups = groups_of(s);
    // no row has more tiles than this
    const long keys = p.window > 0 ? std::min<long>(p.b.max_len, (long)p.window + p.sinks)
                                   : p.b.max_len;
    const long most = (keys + tile_rows<T, HD>() - 1) / tile_rows<T, HD>();
    if (most <= kWholeTiles) p.units = 0;
    const long all = most * p.b.n_rows;
    p.units = (int)std::min<long>(p.units, all);
    p.most_units = (int)std::max<long>(p.units, std::min<long>(4L * p.units, all / kChunk + 1));
    const long pairs = ((long)p.most_units + p.b.n_rows) * s.num_kv_heads;
    const long wgs = (pairs + kXcds - 1) / kXcds * kXcds * (groups / s.num_kv_heads);
    if (all >= 1L << 30 || wgs > (1L << 30) / 256 || (long)p.b.n_rows * s.num_heads > (1L << 30) / 256)
        return hipErrorInvalidValue;
    const dim3 grid((unsigned)wgs);
    const bool reuse = p.kv_mul > p.gb;  // of more than four heads: 3 or 4 of them
    if (p.gb == 1)
        hipLaunchKernelGGL((paged_decode_kernel<T, HD, 1, false>), grid, dim3(256), 0, st, p);
    else if (p.gb == 2)
        hipLaunchKernelGGL((paged_decode_kernel<T, HD, 2, false>), grid, dim3(256), 0, st, p);
    else if (p.gb == 3 && !reuse)
        hipLaunchKernelGGL((paged_decode_kernel<T, HD, 3, false>), grid, dim3(256), 0, st, p);
    else if (p.gb == 3)
        hipLaunchKernelGGL((paged_decode_kernel<T, HD, 3, true>), grid, dim3(256), 0, st, p);
    else if (!reuse)
        hipLaunchKernelGGL((paged_decode_kernel<T, HD, 4, false>), grid, dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((paged_decode_kernel<T, HD, 4, true>), grid, dim3(256), 0, st, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.units) return e;
    hipLaunchKernelGGL((paged_join_kernel<T, HD>), dim3(p.b.n_rows * s.num_heads), dim3(256), 0,
                       st, p);
    return hipGetLastError();
}

template <class T>
hipError_t launch_hd(const Shape& s, const DecodeParams& p, hipStream_t st) {
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

size_t paged_decode_chunks(const Shape& s, int max_rows) {
    return 4 * (size_t)units_of(s, groups_of(s)) + max_rows;
}

hipError_t launch_paged_decode(const Shape& s, const PagedView& b, bool bf16, const float* q,
                               int window, int sinks, float* part_o, float* part_ml, float* out,
                               hipStream_t st) {
    const int gb = gb_of(s.kv_mul);
    const DecodeParams p{b,      q,     out,
                         part_o, part_ml, units_of(s, groups_of(s)), 0,
                         s.num_heads, s.kv_mul, gb,
                         window, sinks, 1.4426950408889634f / sqrtf((float)s.head_dim)};
    return bf16 ? launch_hd<__bf16>(s, p, st) : launch_hd<float>(s, p, st);
}

}  // namespace slm
