// Append (quantise) and read-back kernels of 8-bit pools (THB_KV_E4M3; format
// and page layout in q8.hpp).
//
// Both move head vectors: one lane owns 8 consecutive dims of one vector, the
// lanes of a vector form a segment (a power of two >= head_dim / 8, at least
// 8), and a wavefront holds 64 / segment vectors.
#include <algorithm>
#include <string>

#include "pool.hpp"
#include "q8.hpp"
#include "rope.hpp"

namespace thb {
namespace {

struct Q8Geom {
    uint8_t* k;
    uint8_t* v;
    uint8_t* s;
    const uint32_t* meta;   // row meta at the first row of the call
    const uint32_t* table;  // [seqs * max_pages]
    uint32_t max_pages, pages, seqs, page_shift, head_dim, width, kv_heads, m;
    uint32_t seg_shift;  // log2 of a segment's lanes
};

// Page of a row's token, or false where the row's sequence or page is not the
// pool's (the host checks every row of an eager call; a captured call replays
// with the row meta of its own time).
__device__ inline bool q8_row_page(const Q8Geom& g, uint32_t row, uint32_t& pos, uint32_t& page) {
    pos = g.meta[8 * row];
    const uint32_t seq = g.meta[8 * row + 1];
    if (seq >= g.seqs || (pos >> g.page_shift) >= g.max_pages) return false;
    page = g.table[static_cast<uint64_t>(seq) * g.max_pages + (pos >> g.page_shift)];
    return page < g.pages;
}

// The page's first byte in the planes of codes (head h), and of scales.
__device__ inline uint64_t q8_page_index(const Q8Geom& g, uint32_t h, uint32_t page) {
    return static_cast<uint64_t>(h) * g.pages + page;
}

struct Q8StoreArgs {
    Q8Geom g;
    const void* k_src;  // [m, kv_heads, head_dim]
    const void* v_src;
    uint32_t k_wgs;     // workgroups [0, k_wgs) store K, the others V
    uint32_t rope_on;
    RopeDev rope;
};

// 8 source elements as f32 (exact for the 16-bit types).
template <uint32_t SRC>
__device__ inline void q8_load8(const void* src, uint64_t e, float (&x)[8]) {
    if constexpr (SRC == THB_DT_BF16) {
        const uint4 w = ld_stream16(static_cast<const uint16_t*>(src) + e);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(ws[i] << 16);
            x[2 * i + 1] = __uint_as_float(ws[i] & 0xffff0000u);
        }
    } else {
        load8_f32(SRC, src, e, x);
    }
}

// Largest magnitude's bits over a segment of 1 << seg_shift lanes.
__device__ inline uint32_t q8_seg_max(uint32_t m, uint32_t seg_shift) {
    for (uint32_t i = 0; i < seg_shift; i++) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 1 << i)));
    return m;
}

template <uint32_t SRC>
__global__ __launch_bounds__(256) void q8_store_kernel(Q8StoreArgs a) {
    const Q8Geom& g = a.g;
    const bool is_v = blockIdx.x >= a.k_wgs;
    const uint32_t bid = is_v ? blockIdx.x - a.k_wgs : blockIdx.x;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t seg = lane >> g.seg_shift, u = lane & ((1u << g.seg_shift) - 1u);
    const uint32_t vec = (bid * 4 + (threadIdx.x >> 6)) * (64u >> g.seg_shift) + seg;
    const uint32_t cph = g.head_dim >> 3;
    const bool act = vec < g.m * g.kv_heads && u < cph;
    const uint32_t row = act ? vec / g.kv_heads : 0u, h = act ? vec - row * g.kv_heads : 0u;
    uint32_t pos = 0, page = 0;
    const bool held = act && q8_row_page(g, row, pos, page);
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (act) q8_load8<SRC>(is_v ? a.v_src : a.k_src, static_cast<uint64_t>(vec) * g.head_dim + 8u * u, x);
    if (!is_v && a.rope_on) {  // the rotated key is rounded to the source type first, as thb_rope_rows would leave it
        rope_head_seg(x, act ? u : cph, cph, seg << g.seg_shift, pos, a.rope);
        if constexpr (SRC == THB_DT_F16) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = __uint_as_float(f16_to_f32_bits(f32_to_f16_rne(x[e])));
        }
    }
    const uint32_t b = q8_scale_byte(q8_seg_max(q8_amax8(x), g.seg_shift));
    if (!held) return;
    const uint2 w = q8_encode8(x, b);
    const uint32_t j = pos & ((1u << g.page_shift) - 1u);
    const uint64_t pi = q8_page_index(g, h, page);
    const uint64_t codes = (pi << g.page_shift) * g.width;
    if (!is_v) {
        *reinterpret_cast<uint2*>(g.k + codes + q8_k_off(j, 8u * u, g.width)) = w;
    } else {
        uint8_t* dst = g.v + codes + q8_v_off(j, 8u * u, g.width);
#pragma unroll
        for (int e = 0; e < 8; e++) dst[4 * e] = static_cast<uint8_t>((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
    }
    if (u == 0) g.s[(pi << g.page_shift) * 2u + q8_s_off(j, is_v)] = static_cast<uint8_t>(b);
}

struct Q8LoadArgs {
    Q8Geom g;
    void* k_dst;  // [m, kv_heads, head_dim]
    void* v_dst;
    uint32_t k_wgs;
};

template <uint32_t DT>
__global__ __launch_bounds__(256) void q8_load_kernel(Q8LoadArgs a) {
    const Q8Geom& g = a.g;
    const bool is_v = blockIdx.x >= a.k_wgs;
    const uint32_t bid = is_v ? blockIdx.x - a.k_wgs : blockIdx.x;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t seg = lane >> g.seg_shift, u = lane & ((1u << g.seg_shift) - 1u);
    const uint32_t vec = (bid * 4 + (threadIdx.x >> 6)) * (64u >> g.seg_shift) + seg;
    if (vec >= g.m * g.kv_heads || 8u * u >= g.head_dim) return;
    const uint32_t row = vec / g.kv_heads, h = vec - row * g.kv_heads;
    uint32_t pos, page;
    if (!q8_row_page(g, row, pos, page)) return;
    const uint32_t j = pos & ((1u << g.page_shift) - 1u);
    const uint64_t pi = q8_page_index(g, h, page);
    const uint64_t codes = (pi << g.page_shift) * g.width;
    const float scale = __uint_as_float(static_cast<uint32_t>(g.s[(pi << g.page_shift) * 2u + q8_s_off(j, is_v)]) << 23);
    uint2 w;
    if (!is_v) {
        w = *reinterpret_cast<const uint2*>(g.k + codes + q8_k_off(j, 8u * u, g.width));
    } else {
        const uint8_t* src = g.v + codes + q8_v_off(j, 8u * u, g.width);
        w = make_uint2(0u, 0u);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            w.x |= static_cast<uint32_t>(src[4 * e]) << (8 * e);
            w.y |= static_cast<uint32_t>(src[16 + 4 * e]) << (8 * e);
        }
    }
    float x[8];
    q8_decode8(w, scale, x);
    q8_put8<DT>(is_v ? a.v_dst : a.k_dst, static_cast<uint64_t>(vec) * g.head_dim + 8u * u, x);
}

uint32_t q8_seg_shift(uint32_t head_dim) {
    uint32_t sh = 3;
    while ((1u << sh) < head_dim / 8) sh++;
    return sh;
}

Q8Geom q8_geom(const thb_pool* p, uint32_t layer, const thb_rows* rows, uint32_t row_off, uint32_t m) {
    const LayerGeom& l = p->geom[layer];
    Q8Geom g;
    g.k = p->mem + l.k_off;
    g.v = p->mem + l.v_off;
    g.s = p->mem + l.s_off;
    g.meta = rows->dev + 8 * static_cast<size_t>(row_off);
    g.table = p->table_dev;
    g.max_pages = p->arena.a.max_pages();
    g.pages = p->arena.a.pages();
    g.seqs = p->arena.a.seqs();
    g.page_shift = p->page_shift;
    g.head_dim = l.head_dim;
    g.width = q8_width(l.head_dim);
    g.kv_heads = p->kv_heads;
    g.m = m;
    g.seg_shift = q8_seg_shift(l.head_dim);
    return g;
}

// Workgroups of one operand (K or V) of m rows.
uint32_t q8_wgs(const Q8Geom& g) {
    const uint64_t vecs = static_cast<uint64_t>(g.m) * g.kv_heads, per = 4ull * (64u >> g.seg_shift);
    const uint64_t n = (vecs + per - 1) / per;
    if (vecs > 0x7FFFFFFFull || n > 0x3FFFFFFFull) throw HipError{hipErrorInvalidConfiguration, "append grid too large"};
    return static_cast<uint32_t>(n);
}

}  // namespace

void launch_q8_store(thb_pool* p, uint32_t layer, const void* k_src, const void* v_src, uint32_t src_dtype,
                     const thb_rope* rope, const thb_rows* rows, uint32_t row_off, uint32_t m, hipStream_t s) {
    Q8StoreArgs a;
    a.g = q8_geom(p, layer, rows, row_off, m);
    a.k_src = k_src;
    a.v_src = v_src;
    a.k_wgs = q8_wgs(a.g);
    a.rope_on = rope != nullptr;
    a.rope = rope ? rope_dev(*rope, false) : RopeDev{};
    const dim3 grid(2 * a.k_wgs);
    switch (src_dtype) {
        case THB_DT_F32: hipLaunchKernelGGL(q8_store_kernel<THB_DT_F32>, grid, dim3(256), 0, s, a); break;
        case THB_DT_F16: hipLaunchKernelGGL(q8_store_kernel<THB_DT_F16>, grid, dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL(q8_store_kernel<THB_DT_BF16>, grid, dim3(256), 0, s, a); break;
    }
    THB_HIP(hipGetLastError());
}

void launch_q8_load(thb_pool* p, uint32_t layer, void* k_dst, void* v_dst, uint32_t dst_dtype, const thb_rows* rows,
                    uint32_t row_off, uint32_t m, hipStream_t s) {
    Q8LoadArgs a;
    a.g = q8_geom(p, layer, rows, row_off, m);
    a.k_dst = k_dst;
    a.v_dst = v_dst;
    a.k_wgs = q8_wgs(a.g);
    const dim3 grid(2 * a.k_wgs);
    switch (dst_dtype) {
        case THB_DT_F32: hipLaunchKernelGGL(q8_load_kernel<THB_DT_F32>, grid, dim3(256), 0, s, a); break;
        case THB_DT_F16: hipLaunchKernelGGL(q8_load_kernel<THB_DT_F16>, grid, dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL(q8_load_kernel<THB_DT_BF16>, grid, dim3(256), 0, s, a); break;
    }
    THB_HIP(hipGetLastError());
}

}  // namespace thb
