// Causal attention of runs of rows over a paged cache, on the matrix cores.
//
// A sequence's new rows and the kv_mul query heads of one KV head are packed
// into one list, head fastest: packed row x is row x / kv_mul, head x % kv_mul.
// All of them read the same K and V, so a tile of them is as good as a tile of
// rows of one head, whatever kv_mul is, and short runs fill a tile sooner.
//
// Tiling.  A workgroup has RG groups of 32 packed rows and KSP key splits, a
// wave for each.  A step stages KSP tiles of 32 keys in LDS, row by row: the
// next steps' rows are on their way from their pages while this one is attended
// (straight into LDS where they can, else into registers), and the pages of the
// one after them are being looked up.
// Keys are numbered without the window's gap (Visible of the workgroup's rows).
// Per wave and tile, with v_mfma_f32_32x32x16_bf16:
//   S^T = K . Q^T    A = K rows, B = Q^T (registers): lane (n = l % 32, h = l /
//                    32) ends with the scores of packed row n against keys
//                    8 (r / 4) + 4 h + r % 4 in register r;
//   O^T = V^T . P^T  B = P^T: a lane supplies its own probabilities, so they
//                    never move between lanes; A = V^T with its keys in that
//                    order, by transposing LDS reads.
// Few tiles are split over workgroups as well (find_tile), and joined by a
// second kernel.
//
// Precision.  An f32 value is the sum of three bf16 values (24 bits, each the
// rounded remainder of the ones before).  bf16 pages: q and p are split so, K
// and V are what they are: three products, exact but for f32's rounding of the
// sums.  f32 pages: K and V are split too when they are staged, and of the nine
// products the three below 2^-25 are left out.  q is first scaled by a power of
// two per row, so that values of any size stay within bf16's exponents; the
// scores' scale takes it back.  What cannot be split or must not be multiplied
// makes the workgroup compute its rows again in plain f32 (attend_again): an
// infinity or NaN in a hidden row of V, which leaves one in the sums; where
// values pass through registers any V from 2^64 on, with f32 pages also K, and
// values between 0 and 2^-96, whose remainders run out of exponents.
//
// What bounds it: the matrix cores for long runs, the softmax and the splitting
// between the products next.  Measured, Llama-3-8B shape: 4096 rows, bf16 (137
// GFLOP) 311 us back to back and 392 alone, 442 TFLOP/s in three products each,
// which is the rate of a large library product; behind 2000 rows 630 us alone (436),
// f32 1450 to 1550 (180, six products each); 512 rows bf16 23.8 us.
#include <float.h>
#include <math.h>

#include "paged_common.h"
#include "slm_internal.h"

namespace slm {
namespace {

typedef float v16 __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
typedef unsigned int u2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int KT = 32;  // keys of a tile, packed rows of a wave

struct PrefillParams {
    PagedView b;
    const float* q;
    float* out;
    float* part_o;   // [item][kv head][BM][head_dim]
    float* part_ml;  // [item][kv head][BM][2]
    int units;       // items to aim for; 0: no tile is split
    int num_heads;
    int kv_mul;
    int window;
    int sinks;
    float scale_log2;
};

// Distance of rows in LDS, in 16-byte chunks (16 of which are all banks).  A K
// read takes the same chunk of 32 rows: an odd distance gives 16 neighbouring
// rows all banks.  A V read takes four neighbouring chunks of rows 4 h + (0..3):
// a distance of 4 or 12 modulo 16 spreads four rows over all banks.  As the
// distances are constants, so are the offsets of a lane's reads; slots chosen by
// an exclusive or of row bits meet no conflicts either, but need an address
// register for each read.
constexpr int k_stride(int ch) { return ch | 1; }
constexpr int v_stride(int ch) {
    while (ch % 16 != 4 && ch % 16 != 12) ch += 2;
    return ch;
}

// bf16 planes of a K or V value.
template <class T>
constexpr int planes() {
    return sizeof(T) == 2 ? 1 : 3;
}

// Whether tiles go from the pages straight into LDS: bf16 rows of a power of two
// of chunks.  64 of them are whole rows of one page then, and land side by side,
// so the rows cannot be padded: their chunks are exchanged instead, chunk c of row
// r of a tile lies in slot c ^ swap(r), which the lane that loads it takes into
// account.  Reads pay an exclusive or each; through registers, with their checks
// and stores to LDS, the tiles took 95 of the 445 us of 4096 rows, Llama-3-8B
// shape.
template <class T, int HD>
constexpr bool direct() {
    return sizeof(T) == 2 && HD >= 32 && (HD & (HD - 1)) == 0;
}

// Distinct for rows that are read together: K takes the same chunk of 16
// neighbouring rows, V four chunks (4 d ..) of four rows.
template <int CH>
__device__ __forceinline__ int swap_of(int row) {
    const int four = CH >= 16 ? (row & 3) << 2 : CH == 8 ? (row & 2) << 1 : 0;
    return four | (row >> 2 & 3);
}

// Bytes of one buffer of K and V tiles in LDS, and what a CU has for them.
template <class T, int HD, int KSP>
constexpr int tile_bytes() {
    constexpr int ch = HD / 8;
    return KSP * KT * 16 * planes<T>() *
           (direct<T, HD>() ? 2 * ch : k_stride(ch) + v_stride(ch));
}
constexpr int kLds = 160 * 1024 - 256;

// Two buffers, unless only one lets the CU hold eight waves (where the registers
// do: q and the output of hd 256 leave room for four).  A third one, where it
// fits, gives tiles that go straight into LDS two steps to arrive.
template <class T, int HD, int RG, int KSP>
constexpr int buffers() {
    constexpr int wgs = RG * KSP == 4 && HD <= 128 ? 2 : 1;
    constexpr int most = direct<T, HD>() ? 3 : 2;
    for (int n = most; n > 1; --n)
        if (n * wgs * tile_bytes<T, HD, KSP>() <= kLds) return n;
    return 1;
}

// Waves of a SIMD that the registers are held to: two, unless the tiles in LDS,
// or q and the output alone (hd 256), leave room for one only.
template <class T, int HD, int RG, int KSP>
constexpr int waves_per_simd() {
    if (HD > 128) return 1;
    if (RG * KSP == 8) return 2;
    return 2 * tile_bytes<T, HD, KSP>() <= kLds ? 2 : 1;
}

// The value of lane l ^ 32.
__device__ __forceinline__ float other_half(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float((threadIdx.x & 32) ? a[0] : a[1]);
}

// The largest magnitudes of the values that a thread has staged, and the
// smallest that are not zero; outside() whether they ask for attend_again.
template <class T>
struct Range;
template <>
struct Range<__bf16> {
    us2 top{};  // of the even and the odd values
    __device__ __forceinline__ void add(u4 x) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, x[i] & 0x7FFF7FFFu));
    }
    __device__ __forceinline__ bool outside() const { return max(top[0], top[1]) >= 0x5F80; }
};
template <>
struct Range<float> {
    uint32_t top = 0, low = 0xFFFFFFFFu;  // low: bits less one, so that 0 is the largest
    __device__ __forceinline__ void add(u4 x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = x[i] & 0x7FFFFFFFu;
            top = max(top, u);
            low = min(low, u - 1);
        }
    }
    __device__ __forceinline__ bool outside() const {
        return top >= 0x5F800000u || low < 0x0F800000u - 1;  // 2^64, 2^-96
    }
};

// A tile of packed rows of one sequence, and a chunk of its steps.
struct Tile {
    int seq;     // -1: none
    int index;   // within the sequence
    int row0;    // the sequence's first row of the batch
    int rows;    // and how many it has
    int len;     // as the batch has it
    int chunk;   // within the tile
    int steps;   // of a chunk, at most
    int item0;   // the tile's first chunk, counted over the batch; chunk c is item0 - c
};

constexpr int kUnsplit = 1 << 29;  // steps of a chunk that is the whole tile

// Item (chunk of a tile) `want` of the batch, or with by_tile the first one of
// tile `want`; the last ones first (a sequence's last rows see the most keys).
// With p.units, chunks are so long that about that many make up the batch: a
// sequence of n tiles, none of more than T steps, has n * ceil(T / C) items, C =
// ceil(sum of n * T over the sequences / units).  Every lane of the wave gets
// the same answer.
template <int BM, int KS>
__device__ Tile find_tile(const PrefillParams& p, int want, bool by_tile) {
    const PagedView& b = p.b;
    struct Seq {
        int first, rows, len, tiles, steps;
    };
    const auto seq_of = [&](int s) {
        const int lo = paged_min(paged_max(b.row_start[s], 0), b.n_rows);
        const int rows = paged_min(paged_max(b.row_start[s + 1], lo), b.n_rows) - lo;
        const int len = b.lens[s];
        long long keys = len < 0 || len > b.max_len ? 0 : len;
        if (p.window > 0) keys = min(keys, (long long)p.window + p.sinks + BM / p.kv_mul + 2 + 2 * KT);
        return Seq{lo, rows, len, (int)(((long long)rows * p.kv_mul + BM - 1) / BM),
                   max(1, (int)((keys + KS - 1) / KS))};
    };
    const auto chunk_steps = [&](int total) {
        return p.units ? max(1, (total + p.units - 1) / p.units) : kUnsplit;
    };
    if (b.n_seqs == 1) {  // nothing to look for
        const Seq q = seq_of(0);
        const int c = chunk_steps(q.tiles * q.steps);
        const int k = (q.steps + c - 1) / c, items = q.tiles * k;
        const int at = (by_tile ? q.tiles : items) - 1 - want;
        const int index = by_tile ? at : at / k;
        return Tile{at < 0 ? -1 : 0, index, q.first, q.rows, q.len, by_tile ? 0 : at - index * k, c,
                    items - 1 - index * k};
    }
    // stretches of 64 sequences, the last one first; lane 0 has the last sequence
    const int lane = threadIdx.x & 63;
    const auto mine = [&](int top) {
        const int s = top - 1 - lane;
        return s >= 0 ? seq_of(s) : Seq{0, 0, 0, 0, 1};
    };
    const Seq q0 = mine(b.n_seqs);
    int c = kUnsplit;
    if (p.units) {
        int total = q0.tiles * q0.steps;
        for (int top = b.n_seqs - 64; top > 0; top -= 64) {
            const Seq q = mine(top);
            total += q.tiles * q.steps;
        }
        c = chunk_steps(wave_total(total));
    }
    int before = 0, items_before = 0;
    for (int top = b.n_seqs; top > 0; top -= 64) {
        const Seq q = top == b.n_seqs ? q0 : mine(top);
        const int k = (q.steps + c - 1) / c;
        const int items = wave_upto(q.tiles * k);
        const int cnt = by_tile ? wave_upto(q.tiles) : items;
        const unsigned long long m = __ballot(want < before + cnt);
        if (m) {
            const int l = __ffsll(m) - 1;
            const int at = before + __builtin_amdgcn_readlane(cnt, l) - 1 - want;
            const int kl = __builtin_amdgcn_readlane(k, l);
            const int end = items_before + __builtin_amdgcn_readlane(items, l);
            const int index = __builtin_amdgcn_readfirstlane(by_tile ? at : at / kl);
            return Tile{__builtin_amdgcn_readfirstlane(top - 1 - l),
                        index,
                        __builtin_amdgcn_readlane(q.first, l),
                        __builtin_amdgcn_readlane(q.rows, l),
                        __builtin_amdgcn_readlane(q.len, l),
                        __builtin_amdgcn_readfirstlane(by_tile ? 0 : at - index * kl),
                        __builtin_amdgcn_readfirstlane(c),
                        __builtin_amdgcn_readfirstlane(end - 1 - index * kl)};
        }
        before += __builtin_amdgcn_readlane(cnt, 63);
        items_before += __builtin_amdgcn_readlane(items, 63);
    }
    return Tile{-1, 0, 0, 0, 0, 0, 0, 0};
}

// find_tile's answer in scalar registers (the compiler does not see that every
// lane has the same).
template <int BM, int KS>
__device__ __forceinline__ Tile find_tile_uniform(const PrefillParams& p, int want, bool by_tile) {
    const auto u = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    const Tile t = find_tile<BM, KS>(p, want, by_tile);
    return Tile{u(t.seq), u(t.index), u(t.row0),  u(t.rows),
                u(t.len), u(t.chunk), u(t.steps), u(t.item0)};
}

// Where a tile lies, and the keys that any of its rows sees: Visible of the
// last row, from the first row's window on.
template <int BM, int KS>
struct Span {
    int packed;  // packed rows of the sequence
    int x0;      // the tile's first
    int pos0;    // position of the sequence's first row; of a bad length all are negative
    int pos_first, pos_last;  // of the tile's rows
    bool bad;
    Visible vis;
    int steps;   // of KS keys
    int chunks;
    __device__ __forceinline__ Span(const PrefillParams& p, const Tile& t) : vis(-1, 0, 0) {
        const int len = t.len;
        bad = len < 0 || len > p.b.max_len;
        packed = t.rows * p.kv_mul;
        x0 = t.index * BM;
        pos0 = bad ? -t.rows : len - t.rows;
        pos_first = max(0, pos0 + x0 / p.kv_mul);
        pos_last = pos0 + (min(x0 + BM, packed) - 1) / p.kv_mul;
        vis = Visible(pos_last, 0, 0);
        if (pos_last >= 0 && p.window > 0) {
            vis.lo = max(0, pos_first + 1 - p.window) / KT * KT;
            vis.first = min((min(p.sinks, vis.lo) + KT - 1) / KT * KT, vis.lo);
            vis.count = vis.first + pos_last + 1 - vis.lo;
        }
        steps = (vis.count + KS - 1) / KS;
        chunks = max(1, (steps + t.steps - 1) / t.steps);
    }
};

// Packed rows x, x + step, .. < end of a tile again, one after another by a wave
// that goes through the keys u_beg .. u_end - 1 of vis 64 at a time: scores with
// a key per lane, then the sum with dims over the lanes, in which a key that the
// row does not see has no part.  For the rare tile whose K or V the matrix cores
// cannot take.  The state goes to m, l and o of the row: into out, or the
// partials of row `part` + x.  (Arguments by value: of a reference the caller's
// copy would live in memory, in its hot loop as well.)
template <class T, int HD>
__device__ __noinline__ void attend_again(const PrefillParams p, const Tile tile, int g,
                                          const Visible vis, int u_beg, int u_end, int x, int end,
                                          int step, int pos0, bool bad, bool whole, size_t part) {
    constexpr int NL = (HD + 63) / 64;  // dims of a lane
    const PagedView& b = p.b;
    const int lane = threadIdx.x & 63;
    const T* pages = static_cast<const T*>(b.pages);
    const int32_t* table = b.table + (size_t)tile.seq * b.stride;
    const int slot_mask = (1 << b.ps_shift) - 1;
    for (; x < end; x += step) {
        const int j = x / p.kv_mul;
        const int pos = pos0 + j, pos_out = p.window > 0 ? pos - p.window : -1;
        const size_t at = ((size_t)(tile.row0 + j) * p.num_heads + g * p.kv_mul + x -
                           j * p.kv_mul) * HD;
        float m = -FLT_MAX, l = 0.0f, o[NL] = {};
        for (int u0 = u_beg; u0 < u_end; u0 += 64) {
            const int n = min(64, u_end - u0);
            const int t = vis.row(min(u0 + lane, u_end - 1));
            const bool sees = lane < n && t <= pos && !(t <= pos_out && t >= p.sinks);
            const int page = table[t >> b.ps_shift];
            const bool ok = paged_page_ok(b, page);
            const T* k = pages + paged_at(b, ok ? page : 0, 0, g, t & slot_mask, HD);
            float s = 0.0f;
            for (int d = 0; d < HD; ++d) s = fmaf(p.q[at + d], (float)k[d], s);
            s = !ok ? __builtin_nanf("") : s * p.scale_log2;
            const float mn = fmaxf(m, wave_max(sees ? s : -INFINITY));
            const float alpha = fast_exp2(m - mn);
            const float e = sees ? fast_exp2(s - mn) : 0.0f;
            m = mn;
            l = l * alpha + wave_sum(e);
#pragma unroll
            for (int i = 0; i < NL; ++i) o[i] *= alpha;
            const unsigned long long who = __ballot(sees);
            for (int c = 0; c < n; ++c) {
                if (!(who >> c & 1)) continue;
                const float ec = __shfl(e, c);
                const int tc = vis.row(u0 + c);
                const int pc = table[tc >> b.ps_shift];
                const T* v = pages + paged_at(b, paged_page_ok(b, pc) ? pc : 0, 1, g,
                                              tc & slot_mask, HD);
#pragma unroll
                for (int i = 0; i < NL; ++i) {
                    const int d = min(64 * i + lane, HD - 1);
                    o[i] = fmaf(ec, (float)v[d], o[i]);
                }
            }
        }
        if (!whole && lane == 0) {
            p.part_ml[2 * (part + x)] = m;
            p.part_ml[2 * (part + x) + 1] = l;
        }
#pragma unroll
        for (int i = 0; i < NL; ++i)
            if (64 * i + lane < HD) {
                if (whole)
                    p.out[at + 64 * i + lane] =
                        bad ? __builtin_nanf("") : pos < 0 ? 0.0f : o[i] / l;
                else
                    p.part_o[(part + x) * HD + 64 * i + lane] = o[i];
            }
    }
}

template <class T, int HD, int RG, int KSP>
__global__ __launch_bounds__(64 * RG * KSP, (waves_per_simd<T, HD, RG, KSP>())) void
paged_prefill_kernel(PrefillParams p) {
    constexpr bool BF = sizeof(T) == 2;
    constexpr int NW = RG * KSP, NT = 64 * NW;
    constexpr int BM = 32 * RG;            // packed rows of a workgroup
    constexpr int KS = KSP * KT;           // keys of a step
    constexpr int CH = HD / 8;             // 16-byte chunks of a row's plane
    constexpr int NC = (KS * CH + NT - 1) / NT;  // a thread's chunks of K (and V)
    constexpr bool EXACT = KS * CH % NT == 0;
    constexpr int NL = BF ? 1 : 2;         // 16-byte loads of a chunk's values
    constexpr int NP = planes<T>();
    constexpr int NQ = HD / 16;            // 16-dim steps of K . Q^T
    constexpr int ND = (HD + 31) / 32;     // 32-dim tiles of O^T
    constexpr bool DPAD = HD % 32 != 0;    // the last of them is half empty
    constexpr bool DIRECT = direct<T, HD>();
    constexpr int KST = DIRECT ? CH : k_stride(CH), VST = DIRECT ? CH : v_stride(CH);
    constexpr int MT = KSP == 2 ? (ND + 1) / 2 : ND;  // tiles of O^T that a wave gives away
    // K tiles, then V tiles, NB buffers of NP planes each; at the end the key
    // splits' states
    constexpr int NB = buffers<T, HD, RG, KSP>();
    constexpr int KW = NB * NP * KS * KST, VW = NB * NP * KS * VST;
    constexpr int MERGE = KSP > 1 ? NW * (MT * 256 + 16) : 0;
    __shared__ u4 s_tiles[KW + VW > MERGE ? KW + VW : MERGE];
    u4* const s_k = s_tiles;
    u4* const s_v = s_tiles + KW;

    const PagedView& b = p.b;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, half = lane >> 5;
    const int rg = wave / KSP, ksp = wave % KSP;

    const int g = blockIdx.x % b.kv_heads;
    const int item = blockIdx.x / b.kv_heads;
    const Tile tile = find_tile_uniform<BM, KS>(p, item, false);
    if (tile.seq < 0) return;  // uniform
    const Span<BM, KS> span(p, tile);
    if (tile.chunk >= span.chunks) return;
    const int st_beg = tile.chunk * tile.steps;
    const int st_end = min(span.steps, st_beg + tile.steps);
    const Visible& vis = span.vis;
    const bool bad = span.bad;
    const int packed = span.packed, x0 = span.x0, pos0 = span.pos0;
    const int x = x0 + rg * 32 + n;  // this lane's packed row
    const bool row_ok = x < packed;
    const int j = min(x, packed - 1) / p.kv_mul;
    const int head = g * p.kv_mul + min(x, packed - 1) - j * p.kv_mul;
    const int pos = pos0 + j;  // < 0: an empty row
    const int pos_out = p.window > 0 ? pos - p.window : -1;  // the last row behind the window
    // positions of the wave's rows
    const int xw = x0 + rg * 32;
    const bool wave_ok = xw < packed;
    const int wpos_first = max(0, pos0 + xw / p.kv_mul);
    const int wpos_last = pos0 + (min(xw + 32, packed) - 1) / p.kv_mul;

    const T* pages = static_cast<const T*>(b.pages);
    const int32_t* table = b.table + (size_t)tile.seq * b.stride;
    const int slot_mask = (1 << b.ps_shift) - 1;
    const size_t to_v = ((size_t)b.kv_heads << b.ps_shift) * HD;

    // ---- staging ----
    // Chunk e of a step is chunk e % CH of its row e / CH; a thread has e = tid,
    // tid + NT, ..  Where the 64 chunks of a wave are whole rows of one page
    // (UNI), the page is looked up and the address formed by the scalar unit.
    constexpr bool UNI = CH >= 4 && (CH & (CH - 1)) == 0;
    static_assert(!DIRECT || UNI, "a wave's chunks lie side by side");
    const int pos_last = span.pos_last;
    int page[NC];
    u4 kr[NC][NL], vr[NC][NL];
    // UNI: bit i: the page of chunk i is bad.  Else bit 2i: that, and bit 2i + 1:
    // it lies behind the end.
    unsigned lost = 0;
    const auto key_of = [&](int st, int i) { return st * KS + (tid + i * NT) / CH; };
    const auto first_row = [&](int st, int i) {  // of the wave's chunks i (uniform)
        const int row = (wave * 64 + i * NT) / CH;
        return vis.row(st * KS + row / KT * KT) + row % KT;
    };
    const auto look_up = [&](int st) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if constexpr (UNI)
                page[i] = ((const __attribute__((address_space(4))) int32_t*)
                               table)[min(first_row(st, i), pos_last) >> b.ps_shift];
            else
                page[i] = table[vis.row(min(key_of(st, i), vis.count - 1)) >> b.ps_shift];
        }
    };
    const auto fetch = [&](int st) {
        lost = 0;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const bool ok = paged_page_ok(b, page[i]);
            const T* at;
            if constexpr (UNI) {
                if (!ok) lost |= 1u << i;
                at = pages +
                     paged_at(b, ok ? page[i] : 0, 0, g, first_row(st, i) & slot_mask, HD) +
                     lane * 8;
            } else {
                const int u = key_of(st, i);
                if (!ok) lost |= 1u << (2 * i);
                if (u >= vis.count) lost |= 2u << (2 * i);
                const int t = vis.row(min(u, vis.count - 1));
                at = pages + paged_at(b, ok ? page[i] : 0, 0, g, t & slot_mask, HD) +
                     (tid + i * NT) % CH * 8;
            }
#pragma unroll
            for (int e = 0; e < NL; ++e) {
                kr[i][e] = ((const __attribute__((address_space(1))) u4*)at)[e];
                vr[i][e] = ((const __attribute__((address_space(1))) u4*)(at + to_v))[e];
            }
        }
    };
    // Into LDS.  Rows behind the end are zeros; of a bad page K is NaN, so that
    // the scores of the rows that see it are.
    Range<T> range;
    const auto put = [&](u4* at, int plane, const u4 (&x)[NL]) {
        if constexpr (BF) {
            *at = x[0];
        } else {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(x[e / 4][e % 4]);
            bf8 w[3];
            split8(f, w);
#pragma unroll
            for (int k = 0; k < 3; ++k) at[k * plane] = __builtin_bit_cast(u4, w[k]);
        }
    };
    const auto stage = [&](int st, int buf) {
        const auto set = [&](int i, bool behind) {
            const unsigned w = behind ? 0u : BF ? 0x7FC07FC0u : 0x7FC00000u;
#pragma unroll
            for (int e = 0; e < NL; ++e) {
                kr[i][e] = u4{w, w, w, w};
                vr[i][e] = u4{0, 0, 0, 0};
            }
        };
        if constexpr (UNI) {
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const int t = first_row(st, i);
                if (lost >> i & 1) set(i, false);
                if (t + 64 / CH - 1 > pos_last)  // uniform
                    if (t + lane / CH > pos_last) set(i, true);
            }
        } else if (__any(lost != 0)) {
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (lost & (3u << (2 * i))) set(i, lost & (2u << (2 * i)));
        }
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int e = tid + i * NT, row = e / CH;
            if (!EXACT && row >= KS) break;
#pragma unroll
            for (int h = 0; h < NL; ++h) {
                range.add(vr[i][h]);
                if (!BF) range.add(kr[i][h]);
            }
            put(s_k + (buf * NP * KS + row) * KST + e % CH, KS * KST, kr[i]);
            put(s_v + (buf * NP * KS + row) * VST + e % CH, KS * VST, vr[i]);
        }
    };

    // Straight into LDS: buffer loads, whose range makes zeros of the rows behind
    // the end and of a bad page.  (Inline assembly: the compiler must not make
    // LDS reads of other tiles wait for them.  M0 has the wave's place in LDS.  The
    // load must not issue in the cycle after M0 is written, nor in the five after a
    // vector instruction has written its descriptor.)
    constexpr int AHEAD = NB - 1;  // steps that loads are issued ahead
    static_assert(!DIRECT || (NB >= 2 && (EXACT || NC == 1)), "the waits count a step's loads");
    int src_off[NC];               // where the lane's chunk lies among the wave's
    unsigned lost_of = 0;          // NC bits per step to come: its pages that are bad
    if constexpr (DIRECT) {
#pragma unroll
        for (int i = 0; i < NC; ++i)
            src_off[i] = ((lane & ~(CH - 1)) +
                          (lane % CH ^ swap_of<CH>((wave * 64 + i * NT + lane) / CH))) * 16;
    }
    const auto load_step = [&](int st, int buf, int ahead) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int e0 = wave * 64 + i * NT;
            if (!EXACT && e0 >= KS * CH) break;  // uniform
            const int t = first_row(st, i);
            const bool ok = paged_page_ok(b, page[i]);
            if (!ok) lost_of |= 1u << (ahead * NC + i);
            const int rows = min(64 / CH, max(0, pos_last + 1 - t));
            const T* at = pages + paged_at(b, ok ? page[i] : 0, 0, g, t & slot_mask, HD);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const uint64_t a = reinterpret_cast<uint64_t>(w ? at + to_v : at);
                const u4 r = {(uint32_t)__builtin_amdgcn_readfirstlane((int)a),
                              (uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) & 0xFFFF,
                              (uint32_t)__builtin_amdgcn_readfirstlane(
                                  ok ? rows * HD * (int)sizeof(T) : 0),
                              0x00020000u};
                const unsigned dst = (unsigned)(unsigned long)(
                    __attribute__((address_space(3))) u4*)((w ? s_v : s_k) + buf * KS * CH + e0);
                asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(src_off[i]),
                             "s"(r), "{m0}"(dst) : "memory");
            }
        }
    };
    // The step's tiles are there, for this wave (later ones may be on their way).
    const auto arrived = [&](int st, int buf) {
        if (AHEAD == 2 && st + 1 < st_end)
            asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * NC) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        // K of a bad page is NaN, so that the scores of the rows that see it are
        if (lost_of & ((1u << NC) - 1)) {  // uniform
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (lost_of >> i & 1)
                    s_k[buf * KS * CH + tid + i * NT] =
                        u4{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
        }
        lost_of >>= NC;
    };

    // ---- q ----
    // Lane (n, half) holds dims 16 i + 8 half + (0..7) of packed row n, times
    // log2(e) / sqrt(hd) and a power of two, in three planes.
    float scale;  // what takes the power back: the fused scale and max below are exact
    bf8 qb[NQ][3];
    {
        // the first pages' ids are asked for first, then q, then the first keys
        const bool any = st_beg < st_end;
        if (any) look_up(st_beg);
        const float* src = p.q + ((size_t)(tile.row0 + j) * p.num_heads + head) * HD + 8 * half;
        float xq[NQ][8];
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const float4 a = ld4(src + 16 * i), c = ld4(src + 16 * i + 4);
            const float v[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) xq[i][e] = v[e] * p.scale_log2;
        }
        if (any) {
            if constexpr (DIRECT)
                load_step(st_beg, 0, 0);
            else
                fetch(st_beg);
            if (st_beg + 1 < st_end) look_up(st_beg + 1);
        }
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(xq[i][e]));
        top = fmaxf(top, other_half(top));
        // largest magnitude in [2^-10, 2^-9): sums of 256 products with any bf16 K
        // stay finite
        int ex = 0;
        if (top > 0.0f && top < INFINITY) {
            (void)frexpf(top, &ex);
            ex += 9;
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) xq[i][e] = ldexpf(xq[i][e], -ex);
            split8(xq[i], qb[i]);
        }
        // (never 0 or infinite: hidden scores must stay -inf, scores of 0 must stay 0)
        scale = ldexpf(1.0f, min(max(ex, -126), 127));
    }

    v16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = v16{};
    float m = -FLT_MAX, l = 0.0f;  // finite m: a row that has seen no key yet needs no guard

    // ---- one tile of the wave ----
    // The products of planes (K or V, q or p), small ones first.
    constexpr int NPR = BF ? 3 : 6;
    constexpr int PA[6] = {BF ? 0 : 2, 0, BF ? 0 : 1, 1, 0, 0};
    constexpr int PB[6] = {BF ? 2 : 0, BF ? 1 : 2, BF ? 0 : 1, 0, 1, 0};
    const auto attend = [&](int buf, int u0) {
        const u4* sk = s_k + (buf * NP * KS + ksp * KT) * KST;
        const u4* sv = s_v + (buf * NP * KS + ksp * KT) * VST;
        // DIRECT: bytes from there to the lane's chunks 0 (a tile's first byte has
        // the low bits 0, so the exclusive ors below may follow the sums)
        const unsigned ka = (unsigned)(n * CH + (half ^ swap_of<CH>(n))) * 16;
        const int vrow = 4 * half + (lane >> 2 & 3);
        const unsigned va =
            (unsigned)(vrow * CH + ((lane >> 3 & 2) + (lane >> 1 & 1) ^ swap_of<CH>(vrow))) * 16 +
            8 * (lane & 1);
        v16 s = v16{};
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            bf8 kf[NP];
#pragma unroll
            for (int k = 0; k < NP; ++k)
                kf[k] = __builtin_bit_cast(
                    bf8, DIRECT ? *reinterpret_cast<const u4*>(reinterpret_cast<const char*>(sk) +
                                                               (ka ^ 32u * i))
                                : sk[k * KS * KST + n * KST + 2 * i + half]);
#pragma unroll
            for (int e = 0; e < NPR; ++e)
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[PA[e]], qb[i][PB[e]], s, 0, 0, 0);
        }
        // the tile's rows are t0 .. t0 + 31; some behind the end (t > every pos)
        const int t0 = vis.row(u0);
        if (t0 + KT - 1 > wpos_first ||
            (p.window > 0 && t0 <= wpos_last - p.window && t0 + KT > p.sinks)) {  // uniform
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int t = t0 + 8 * (r / 4) + 4 * half + r % 4;
                const bool hide = (t > pos) | ((t <= pos_out) & (t >= p.sinks));
                s[r] = hide ? -INFINITY : s[r];
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
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            bf8 pf[3];
            const float xs[8] = {s[8 * ks],     s[8 * ks + 1], s[8 * ks + 2], s[8 * ks + 3],
                                 s[8 * ks + 4], s[8 * ks + 5], s[8 * ks + 6], s[8 * ks + 7]};
            split8(xs, pf);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                // 16 lanes read a 4 x 16 block row by row and get it column by
                // column; dims behind HD repeat others
                const int dim = DPAD && d == ND - 1 ? 4 * (lane & 3)
                                                    : 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
                bf8 vf[NP];
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    s4 w[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int row = 16 * ks + 8 * c + 4 * half + ((lane >> 2) & 3);
                        const short* at =
                            DIRECT ? reinterpret_cast<const short*>(
                                         reinterpret_cast<const char*>(sv) +
                                         (16 * ks + 8 * c) * CH * 16 +
                                         (va ^ (unsigned)(4 * d ^ 2 * c) * 16))
                                   : reinterpret_cast<const short*>(sv + k * KS * VST + row * VST) +
                                         32 * d + dim;
                        w[c] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s4*)(at));
                    }
                    const u2 w0 = __builtin_bit_cast(u2, w[0]), w1 = __builtin_bit_cast(u2, w[1]);
                    vf[k] = __builtin_bit_cast(bf8, u4{w0[0], w0[1], w1[0], w1[1]});
                }
#pragma unroll
                for (int e = 0; e < NPR; ++e)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[PA[e]], pf[PB[e]], o[d], 0, 0,
                                                                   0);
            }
        }
    };

    // ---- the steps ----
    // (a wave whose rows are all empty or in front of a tile has nothing to do
    // there)
    const auto attend_step = [&](int st, int buf) {
        const int u0 = st * KS + ksp * KT;
        if (wave_ok && u0 < vis.count && vis.row(u0) <= wpos_last) attend(buf, u0);
    };
    bool outside;
    if constexpr (DIRECT) {
        if (AHEAD == 2 && st_beg + 1 < st_end) {
            load_step(st_beg + 1, 1, 1);
            if (st_beg + 2 < st_end) look_up(st_beg + 2);
        }
        int buf = 0;
        for (int st = st_beg; st < st_end; ++st) {
            arrived(st, buf);
            __syncthreads();
            // every wave is done with the buffer of the step before
            if (st + AHEAD < st_end) {
                load_step(st + AHEAD, buf == 0 ? NB - 1 : buf - 1, AHEAD - 1);
                if (st + AHEAD + 1 < st_end) look_up(st + AHEAD + 1);
            }
            attend_step(st, buf);
            buf = buf == NB - 1 ? 0 : buf + 1;
        }
        // what must not be multiplied has left an infinity or NaN
        float x = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) x = fmaf(o[d][r], 0.0f, x);
        outside = x != x;
    } else {
        for (int st = st_beg; st < st_end; ++st) {
            const int buf = NB == 2 ? st & 1 : 0;
            stage(st, buf);
            if (st + 1 < st_end) {
                fetch(st + 1);
                if (st + 2 < st_end) look_up(st + 2);
            }
            __syncthreads();
            attend_step(st, buf);
            if (NB == 1) __syncthreads();
        }
        outside = range.outside();
    }
    l += other_half(l);
    const bool redo = __syncthreads_or(outside);  // (and every wave is done with the tiles)

    // ---- key splits ----
    if constexpr (KSP > 1) {
        // Every wave scales its state to the row's max over the splits.  Split k
        // sums tiles k, k + KSP, .. of O^T, which the others leave it in the
        // bytes of the K and V tiles.
        float* const s_o = reinterpret_cast<float*>(s_tiles);
        float* const s_ml = s_o + NW * MT * 1024;
        const auto slot = [&](int w, int d) {
            return s_o + (w * MT + (KSP == 2 ? d / 2 : d)) * 1024 + lane;
        };
        if (half == 0) {
            s_ml[wave * 64 + n] = m;
            s_ml[wave * 64 + 32 + n] = l;
        }
        __syncthreads();
        float top = m;
#pragma unroll
        for (int k = 0; k < KSP; ++k) top = fmaxf(top, s_ml[(rg * KSP + k) * 64 + n]);
        const float e = fast_exp2(m - top);
        m = top;
        l = 0.0f;
#pragma unroll
        for (int k = 0; k < KSP; ++k)
            l += s_ml[(rg * KSP + k) * 64 + 32 + n] *
                 fast_exp2(s_ml[(rg * KSP + k) * 64 + n] - top);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            o[d] *= e;
            if (d % KSP != ksp)
#pragma unroll
                for (int r = 0; r < 16; ++r) slot(wave, d)[64 * r] = o[d][r];
        }
        __syncthreads();
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if (d % KSP != ksp) continue;  // uniform
#pragma unroll
            for (int k = 1; k < KSP; ++k) {
                const int w = rg * KSP + (ksp + k) % KSP;
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] += slot(w, d)[64 * r];
            }
        }
    }

    // ---- the output ----
    const bool whole = span.chunks == 1;
    const size_t part = ((size_t)item * b.kv_heads + g) * BM;  // the tile's first partial row
    if (redo) {  // uniform
        if (wave_ok)
            attend_again<T, HD>(p, tile, g, vis, st_beg * KS, min(vis.count, st_end * KS),
                                xw + ksp, min(xw + 32, packed), KSP, pos0, bad, whole, part - x0);
        return;
    }
    if (!row_ok) return;
    float* dst = p.out + ((size_t)(tile.row0 + j) * p.num_heads + head) * HD;
    // an empty row gives zeros, one of a bad length NaN
    float inv = bad ? __builtin_nanf("") : pos < 0 ? 0.0f : 1.0f / l;
    if (!whole) {  // uniform
        const size_t r = part + rg * 32 + n;
        if (half == 0 && ksp == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * r) = make_float2(m, l);
        dst = p.part_o + r * HD;
        inv = 1.0f;
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        if (d % KSP != ksp) continue;
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int dim = 32 * d + 8 * (r / 4) + 4 * half;
            if (DPAD && d == ND - 1 && r >= 8) break;
            *reinterpret_cast<float4*>(dst + dim) = make_float4(o[d][r] * inv, o[d][r + 1] * inv,
                                                                o[d][r + 2] * inv, o[d][r + 3] * inv);
        }
    }
}

// Joins the chunks of a tile for one KV head: four dims of a packed row per
// thread.  Bound by its launch and two round trips to memory: 4.2 us.
template <int HD, int BM, int KS>
__global__ __launch_bounds__(kThreads) void paged_prefill_join_kernel(PrefillParams p) {
    constexpr int PARTS = (BM * HD / 4 + kThreads - 1) / kThreads;  // workgroups of a tile
    const PagedView& b = p.b;
    const int part = blockIdx.x % PARTS, g = blockIdx.x / PARTS % b.kv_heads;
    const Tile tile =
        find_tile_uniform<BM, KS>(p, blockIdx.x / (PARTS * b.kv_heads), true);
    if (tile.seq < 0) return;
    const Span<BM, KS> span(p, tile);
    if (span.chunks == 1) return;  // written by its workgroup
    const int e = part * kThreads + threadIdx.x;
    const int row = e / (HD / 4), dim = e % (HD / 4) * 4;
    const int x = span.x0 + row;
    if (row >= BM || x >= span.packed) return;
    const size_t first = ((size_t)tile.item0 * b.kv_heads + g) * BM + row;
    const size_t back = (size_t)b.kv_heads * BM;  // from a chunk to the one before
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
    float m = -FLT_MAX, l = 0.0f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    // eight chunks in flight; those behind the last repeat it with weight 0
    for (int c0 = 0; c0 < span.chunks; c0 += 8) {
        float2 y[8];
        float4 z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const size_t r = first - min(c0 + i, span.chunks - 1) * back;
            y[i] = ml[r];
            z[i] = ld4(p.part_o + r * HD + dim);
        }
        float mn = m;
#pragma unroll
        for (int i = 0; i < 8; ++i) mn = fmaxf(mn, y[i].x);
        const float a = fast_exp2(m - mn);
        m = mn;
        l *= a;
        o.x *= a, o.y *= a, o.z *= a, o.w *= a;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (c0 + i >= span.chunks) break;
            const float w = fast_exp2(y[i].x - m);
            l += w * y[i].y;
            o.x = fmaf(w, z[i].x, o.x);
            o.y = fmaf(w, z[i].y, o.y);
            o.z = fmaf(w, z[i].z, o.z);
            o.w = fmaf(w, z[i].w, o.w);
        }
    }
    const int j = x / p.kv_mul;
    const int head = g * p.kv_mul + x - j * p.kv_mul;
    const float inv = span.pos0 + j < 0 ? 0.0f : 1.0f / l;  // an empty row gives zeros
    *reinterpret_cast<float4*>(p.out + ((size_t)(tile.row0 + j) * p.num_heads + head) * HD + dim) =
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// At most this many tiles of BM packed rows, whatever the rows' division among
// the sequences.
long tiles_bound(const PagedView& b, int kv_mul, int bm) {
    return ((long)b.n_rows * kv_mul + (long)b.n_seqs * (bm - 1)) / bm;
}

// No row sees more keys than this.
long keys_bound(const PrefillParams& p) {
    const long w = (long)p.window + p.sinks;
    return p.window > 0 && w < p.b.max_len ? w : p.b.max_len;
}

template <class T, int HD, int RG, int KSP>
hipError_t launch_k(const Shape& s, PrefillParams p, hipStream_t st) {
    constexpr int BM = 32 * RG, KS = KSP * KT, NT = 64 * RG * KSP;
    static_assert(tile_bytes<T, HD, KSP>() <= kLds, "the tiles fit a CU");
    const long tiles = tiles_bound(p.b, s.kv_mul, BM);
    // Tiles that leave CUs empty are split into as many chunks as still run side
    // by side, if that takes two steps or more off the longest (one sequence, hd 64
    // f32, 128 rows behind 350: 13.2 us, 19.5 with a limit of four steps; bf16, 64
    // rows alone: 7.4 us, 9.5 with one of one and a half).
    const long ns = s.cus / (tiles * s.num_kv_heads);
    const long steps = (keys_bound(p) + KS - 1) / KS;
    p.units = ns >= 2 && steps * (ns - 1) >= 2 * ns ? (int)(ns * tiles) : 0;
    // (the plan's sums are 32-bit, also of row starts that overlap)
    if (tiles * steps * p.b.n_seqs >= 1L << 30) p.units = 0;
    const long wgs = (tiles + p.units) * s.num_kv_heads;
    if (wgs >= (1L << 32) / NT) return hipErrorInvalidValue;
    hipLaunchKernelGGL((paged_prefill_kernel<T, HD, RG, KSP>), dim3((unsigned)wgs), dim3(NT), 0, st,
                       p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.units) return e;
    constexpr int parts = (BM * HD / 4 + kThreads - 1) / kThreads;
    hipLaunchKernelGGL((paged_prefill_join_kernel<HD, BM, KS>),
                       dim3((unsigned)(tiles * s.num_kv_heads * parts)), dim3(kThreads), 0, st, p);
    return hipGetLastError();
}

// Groups of packed rows and key splits of a workgroup, by wgs, the workgroups
// that 128-row tiles make, and the keys of the longest row.  Four groups share
// what is staged; key splits put eight waves on a CU that would have four and
// shorten the longest workgroup, and fewer groups make more workgroups, where
// there are few, or where those of 128 rows would leave some CUs without one; a
// split over workgroups (launch_k) costs a second launch, but needs no merge in
// LDS.  Measured for one sequence, page 32, 256 CUs (us):
//   hd 128  4 x 1 / 4 x 2 / 2 x 2        bf16                f32
//     16 rows (wgs 8)                     7.4 / 10.3 / 9.4    9.4 / 12.5 / 12.2
//     256 rows (wgs 64)                   18.4 / 20.6 / 16.8  23.2 / 25.4 / 22.3
//     512 rows (wgs 128)                  27.4 / 27.0 / 23.8  44.8 / 40.3 / 46.4
//     768 rows (wgs 192)                  44.3 / 36.2 / 33.8  96 / 77 / 66
//     64 rows behind 2000 (wgs 16)        25.9 / 26.4 / 24.8  37.0 / 35.8 / 38.5
//     256 rows behind 2000 (wgs 64)       44.5 / 41.8 / 49.8  83 / 71 / 101
//     2048 rows behind 2000 (wgs 512)     260 / 249 / 271     584 / 586 / 962
//     4096 rows behind 2000 (wgs 1024)    629 / 655 / 711     1523 / 1533 / 2529
//     16 rows of 8 heads behind 2000 (2)  32.1 / 24.9 / 23.7  34.8 / 29.2 / 26.7
//   hd 64   4 x 2 / 2 x 4 / 1 x 8 (f32: 1 x 4)
//     256 rows (wgs 18)                   12.6 / 10.1 / 9.3   13.5 / 13.5 / 12.5
//     1024 rows (wgs 72)                  20.3 / 19.1 / 17.1  26.9 / 33.5 / 33.3
//     1536 rows (wgs 108)                 28.3 / 25.1 / 26.6  42.2 / 46.8 / 51.4
//     2048 rows (wgs 144)                 50.6 / 30.9 / 40.7  89 / 60 / 87
//     64 rows behind 2000 (wgs 6)         22.3 / 17.4 / 14.9  23.5 / 18.8 / 17.7
//     256 rows behind 2000 (wgs 18)       20.3 / 17.1 / 17.3  23.4 / 22.6 / 30.6
//     1024 rows behind 2000 (wgs 72)      35.6 / 42.4 / 48.8  53.7 / 86.8 / 132
//   hd 256  4 x 1 / 2 x 2
//     512 rows (wgs 16)                   29.7 / 24.2
//     1024 rows behind 2000 (wgs 32)      59.2 / 62.5
template <class T, int HD>
hipError_t launch_t(const Shape& s, const PrefillParams& p, hipStream_t st) {
    constexpr bool BF = sizeof(T) == 2;
    const long wgs = tiles_bound(p.b, s.kv_mul, 128) * s.num_kv_heads;
    const long keys = keys_bound(p), cus = s.cus;
    if constexpr (HD > 128) {
        if constexpr (BF)
            if (keys > 128 && wgs <= cus / (keys <= 1024 ? 8 : 16))
                return launch_k<T, HD, 2, 2>(s, p, st);
    } else if constexpr (HD > 64) {
        if (keys > 32) {
            // whole sequences, whose last rows see twice the average: by smaller
            // workgroups where less than a round of large ones would wait for them
            const bool uneven = wgs > cus / 2 && wgs < cus && keys <= 1536 &&
                                4 * keys * p.b.n_seqs <= 5L * p.b.n_rows;
            const bool few = BF ? wgs <= cus / (keys <= 512 ? 2 : 16)
                                : wgs <= cus / (keys <= 256 ? 4 : 32);
            if (few || uneven)
                return launch_k<T, HD, 2, 2>(s, p, st);
            if (wgs < 3 * cus) return launch_k<T, HD, 4, 2>(s, p, st);
        }
    } else if (keys > 64) {
        constexpr bool k8 = tile_bytes<T, HD, 8>() <= kLds;  // or four splits
        if (wgs <= (keys > 2048 ? cus / (k8 ? 16 : 32) : k8 ? cus * 3 / 8 : cus / 8))
            return launch_k<T, HD, 1, k8 ? 8 : 4>(s, p, st);
        if (wgs <= cus / 8 || (wgs > cus * (BF ? 3 : 4) / 8 && wgs <= cus * 3 / 4))
            return launch_k<T, HD, 2, 4>(s, p, st);
        if (wgs < 3 * cus) return launch_k<T, HD, 4, 2>(s, p, st);
    }
    return launch_k<T, HD, 4, 1>(s, p, st);
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

// Items times KV heads are at most tiles (fewer than CUs where they are split)
// and the CUs again; a tile has at most 128 rows.
size_t paged_prefill_part_rows(const Shape& s) { return (size_t)2 * s.cus * 128; }

hipError_t launch_paged_prefill(const Shape& s, const PagedView& b, bool bf16, const float* q,
                                int window, int sinks, float* part_o, float* part_ml, float* out,
                                hipStream_t st) {
    const PrefillParams p{b,      q,     out, part_o, part_ml, 0, s.num_heads, s.kv_mul, window,
                          sinks, 1.4426950408889634f / sqrtf((float)s.head_dim)};
    return bf16 ? launch_hd<__bf16>(s, p, st) : launch_hd<float>(s, p, st);
}

}  // namespace slm
