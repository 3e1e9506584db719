// Rows of a batch into the paged cache: optional norm of each q and k head,
// rotation at the row's position, and the store of K and V into their page, in
// one pass.
//
// x' = x * (1 / sqrt(mean(x^2) + eps)) * w per head, then apply_rope_cached
// (transformer.rs:178-194) with every product and sum rounded on its own, as
// in rope_append.hip: without norms f32 pages get slm_kv_append_dev's bits.
//
// What bounds it: each value is read once and written once, 3 to 7 flops in
// between.  A head lies in the 16-byte loads of one lane group (the next power
// of two of head_dim / 4 lanes), so the norm's sum is a few lane swaps and
// nothing goes through LDS.  A workgroup works on one row: its sequence and
// position are found once per wave, by one load and a ballot for up to 63
// sequences.  Measured: 5390 rows of the Llama-3-8B shape into bf16 pages with both
// norms (243 MB) 48 us back to back, 5.05 TB/s, a large copy's rate; one row 2.9 us.
#include "paged_common.h"
#include "slm_internal.h"

namespace slm {
namespace {

typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void store4(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }
__device__ __forceinline__ void store4(__bf16* p, float4 x) {
    *reinterpret_cast<bf4*>(p) = __builtin_convertvector(f4{x.x, x.y, x.z, x.w}, bf4);
}

struct AppendParams {
    PagedView b;
    const float* q;  // nullptr: no q heads
    const float* k;
    const float* v;
    const float* q_norm;  // nullptr: no norm
    const float* k_norm;
    const float* cos_t;
    const float* sin_t;
    float* q_out;
    float eps;
    int q_heads;  // 0 without q
    int row0;     // first row of this launch
};

// Lanes of one head: a power of two, at most a wave.
template <int HD>
constexpr int head_lanes() {
    int l = 1;
    while (l < HD / 4) l *= 2;
    return l;
}

constexpr int kThreads = 256;

template <class T, int HD>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(AppendParams p, int blocks_per_row) {
    constexpr int LPH = head_lanes<HD>();
    const PagedView& b = p.b;
    const int row_here = blockIdx.x / blocks_per_row;
    const int part = blockIdx.x - row_here * blocks_per_row;
    const int row = p.row0 + row_here;
    const int c = threadIdx.x % LPH;  // this lane's dims: 4c .. 4c + 3
    const int item = part * (kThreads / LPH) + threadIdx.x / LPH;
    const bool active = item < p.q_heads + 2 * b.kv_heads && c < HD / 4;

    // the head's values are on their way while the row is looked up
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), w = x;
    const int h = item - p.q_heads;  // < 0: a q head; then K heads, then V heads
    const bool is_v = h >= b.kv_heads;
    const float* norm = h < 0 ? p.q_norm : is_v ? nullptr : p.k_norm;
    if (active) {
        const float* src = h < 0 ? p.q + ((size_t)row * p.q_heads + item) * HD
                                 : (is_v ? p.v + ((size_t)row * b.kv_heads + h - b.kv_heads) * HD
                                         : p.k + ((size_t)row * b.kv_heads + h) * HD);
        x = ld4(src + 4 * c);
        if (norm) w = ld4(norm + 4 * c);
    }
    const PagedRow r = paged_row_wave(b, row);
    if (r.seq < 0 || (r.pos < 0 && !r.bad)) return;  // uniform: no row, or an empty one
    if (r.bad) {
        if (active && h < 0) {
            const float n = __builtin_nanf("");
            store4(p.q_out + ((size_t)row * p.q_heads + item) * HD + 4 * c,
                   make_float4(n, n, n, n));
        }
        return;
    }
    const int page = b.table[(size_t)r.seq * b.stride + (r.pos >> b.ps_shift)];
    float2 cs = make_float2(1.f, 1.f), sn = make_float2(0.f, 0.f);
    if (active && !is_v) {
        const size_t t = (size_t)r.pos * (HD / 2) + 2 * c;
        cs = *reinterpret_cast<const float2*>(p.cos_t + t);
        sn = *reinterpret_cast<const float2*>(p.sin_t + t);
    }
    if (p.q_norm || p.k_norm) {  // uniform: the lane swaps need every lane
        float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w;
        ss = group_sum<LPH>(ss);
        if (norm) {
            const float rms = 1.0f / sqrtf(ss * (1.0f / HD) + p.eps);
            x.x = x.x * rms * w.x;
            x.y = x.y * rms * w.y;
            x.z = x.z * rms * w.z;
            x.w = x.w * rms * w.w;
        }
    }
    if (!active) return;
    if (!is_v) x = rope4_exact(x, cs, sn);
    if (h < 0) {
        store4(p.q_out + ((size_t)row * p.q_heads + item) * HD + 4 * c, x);
    } else if (paged_page_ok(b, page)) {
        T* dst = static_cast<T*>(b.pages) + paged_at(b, page, is_v, is_v ? h - b.kv_heads : h,
                                                     r.pos & ((1 << b.ps_shift) - 1), HD);
        store4(dst + 4 * c, x);
    }
}

template <class T, int HD>
hipError_t launch_t(AppendParams p, hipStream_t st) {
    constexpr int per_block = kThreads / head_lanes<HD>();
    const int bpr = (p.q_heads + 2 * p.b.kv_heads + per_block - 1) / per_block;
    // a launch has fewer than 2^32 threads
    const int step = (1 << 30) / kThreads / bpr;
    for (p.row0 = 0; p.row0 < p.b.n_rows; p.row0 += step) {
        const int rows = p.b.n_rows - p.row0 < step ? p.b.n_rows - p.row0 : step;
        hipLaunchKernelGGL((paged_append_kernel<T, HD>), dim3((unsigned)bpr * (unsigned)rows),
                           dim3(kThreads), 0, st, p, bpr);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        if (rows == p.b.n_rows - p.row0) break;  // row0 + step could pass 2^31
    }
    return hipSuccess;
}

template <class T>
hipError_t launch_hd(int head_dim, const AppendParams& p, hipStream_t st) {
    switch (head_dim) {
        case 16: return launch_t<T, 16>(p, st);
        case 32: return launch_t<T, 32>(p, st);
        case 48: return launch_t<T, 48>(p, st);
        case 64: return launch_t<T, 64>(p, st);
        case 96: return launch_t<T, 96>(p, st);
        case 128: return launch_t<T, 128>(p, st);
        case 256: return launch_t<T, 256>(p, st);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_paged_append(const Shape& s, const PagedView& b, bool bf16, const float* q,
                               const float* k, const float* v, const float* q_norm,
                               const float* k_norm, float eps, const float* cos_t,
                               const float* sin_t, float* q_out, hipStream_t st) {
    const AppendParams p{b,     q,     k,   v,     q_norm, k_norm, cos_t,
                         sin_t, q_out, eps, q ? s.num_heads : 0, 0};
    return bf16 ? launch_hd<__bf16>(s.head_dim, p, st) : launch_hd<float>(s.head_dim, p, st);
}

}  // namespace slm
