// Append (quantise) and read-back kernels of 8-bit pools (THB_KV_E4M3; format
// and page layout in q8.hpp).
//
// Both move head vectors: one lane owns 8 consecutive dims of one vector (or of 4,
// of consecutive rows), the lanes of a vector form a segment (a power of two >=
// head_dim / 8, at least 8), and a wavefront holds 64 / segment of them.
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

// Rows of a segment: RB consecutive ones of one head.  Groups of RB rows start
// where slots do that are a multiple of RB, in the chunk that the call begins with
// or, if its first two rows are no chunk, ends with (64 decode rows and 8 chunks of
// 512: 10 us to append, 15 to read back, 20 with groups that start inside the
// chunks' groups of slots, as those of chunks elsewhere in a call may).
template <uint32_t RB>
struct Q8Rows {
    uint32_t u, h, row0;          // the lane's unit of 8 dims, head, first row (may be "negative")
    uint32_t on, held;            // bits: rows of the call; of those, rows whose page is the pool's
    uint32_t pos[RB], page[RB];
    bool run;                     // RB whole rows, at RB consecutive slots from a multiple of RB

    __device__ Q8Rows(const Q8Geom& g, uint32_t bid) {
        const uint32_t lane = threadIdx.x & 63u;
        u = lane & ((1u << g.seg_shift) - 1u);
        const uint32_t i = (bid * 4 + (threadIdx.x >> 6)) * (64u >> g.seg_shift) + (lane >> g.seg_shift);
        const uint32_t gr = i / g.kv_heads;
        h = i - gr * g.kv_heads;
        row0 = gr * RB;
        if (RB > 1 && g.m > 1) {
            const bool first = g.meta[8] == g.meta[0] + 1u;
            const uint32_t r = first ? 0u : g.m - 1u;
            row0 -= (g.meta[8 * r] - r) & (RB - 1u);
        }
        on = held = 0;
        run = RB > 1;
#pragma unroll
        for (uint32_t r = 0; r < RB; r++) {
            pos[r] = page[r] = 0;
            if (row0 + r < g.m) {  // (a row before the first is a large number)
                on |= 1u << r;
                held |= q8_row_page(g, row0 + r, pos[r], page[r]) ? 1u << r : 0u;
            }
            run = run && pos[r] == (pos[0] | r) && page[r] == page[0];
        }
        run = run && held == (1u << RB) - 1u && (pos[0] & (RB - 1u)) == 0;
    }
};

// RB: rows a lane handles.  A byte of V per slot and dim is a store of its own
// where a token comes alone; RB = 4 tokens of consecutive slots fill the words of
// their 4-slot groups: 16-byte stores of V, and of K between two lanes that
// hold the two halves of a slot's 16 bytes.  Bound by its bytes: 4096 bf16 rows of
// 8 KV heads of 128, 25 MB, 10.1 us, reading them back 9.2; the pair of calls 30,
// which is their host time (with byte stores 35).
template <uint32_t SRC, uint32_t RB>
__global__ __launch_bounds__(256) void q8_store_kernel(Q8StoreArgs a) {
    const Q8Geom& g = a.g;
    const bool is_v = blockIdx.x >= a.k_wgs;
    const Q8Rows<RB> R(g, is_v ? blockIdx.x - a.k_wgs : blockIdx.x);
    const uint32_t u = R.u, cph = g.head_dim >> 3;
    float x[RB][8];
#pragma unroll
    for (uint32_t r = 0; r < RB; r++) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[r][e] = 0.0f;
        if ((R.on >> r & 1u) && u < cph)
            q8_load8<SRC>(is_v ? a.v_src : a.k_src,
                          (static_cast<uint64_t>(R.row0 + r) * g.kv_heads + R.h) * g.head_dim + 8u * u, x[r]);
    }
    uint2 w[RB];
    uint32_t b[RB];
#pragma unroll
    for (uint32_t r = 0; r < RB; r++) {
        if (!is_v && a.rope_on) {  // the rotated key is rounded to the source type first, as thb_rope_rows would leave it
            rope_head_seg(x[r], (R.on >> r & 1u) && u < cph ? u : cph, cph, (threadIdx.x & 63u) - u, R.pos[r], a.rope);
            if constexpr (SRC == THB_DT_F16) {
#pragma unroll
                for (int e = 0; e < 8; e++) x[r][e] = __uint_as_float(f16_to_f32_bits(f32_to_f16_rne(x[r][e])));
            }
        }
        b[r] = q8_scale_byte(q8_seg_max(q8_amax8(x[r]), g.seg_shift));
        w[r] = q8_encode8(x[r], b[r]);
    }
    if constexpr (RB == 4) {
        if (R.run) {
            const uint32_t j = R.pos[0] & ((1u << g.page_shift) - 1u);
            const uint64_t pi = q8_page_index(g, R.h, R.page[0]);
            const uint64_t codes = (pi << g.page_shift) * g.width;
            if (u == 0)
                *reinterpret_cast<uint32_t*>(g.s + (pi << g.page_shift) * 2u + q8_s_off(j, is_v)) =
                    b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
            if (is_v) {
                if (u >= cph) return;
                u32x4 t[2];  // by dim, the 4 slots' codes
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    const uint32_t w0 = d ? w[0].y : w[0].x, w1 = d ? w[1].y : w[1].x;
                    const uint32_t w2 = d ? w[2].y : w[2].x, w3 = d ? w[3].y : w[3].x;
                    const uint32_t a01 = __builtin_amdgcn_perm(w1, w0, 0x05010400), b01 = __builtin_amdgcn_perm(w1, w0, 0x07030602);
                    const uint32_t a23 = __builtin_amdgcn_perm(w3, w2, 0x05010400), b23 = __builtin_amdgcn_perm(w3, w2, 0x07030602);
                    t[d] = u32x4{__builtin_amdgcn_perm(a23, a01, 0x05040100), __builtin_amdgcn_perm(a23, a01, 0x07060302),
                                 __builtin_amdgcn_perm(b23, b01, 0x05040100), __builtin_amdgcn_perm(b23, b01, 0x07060302)};
                }
                u32x4* dst = reinterpret_cast<u32x4*>(g.v + codes + q8_v_off(j, 8u * u, g.width));
                dst[0] = t[0];
                dst[1] = t[1];
                return;
            }
            // Units u and u + 4 of a 64-dim block hold a slot's 16 bytes: the first lane
            // takes rows 0 and 1, the second 2 and 3.  (A block's padding, where
            // head_dim ends inside it, gets the zero codes it has.)
            const bool hi = (u & 4u) != 0;
            u32x4 o[2];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const uint2 give = hi ? w[r] : w[r + 2], own = hi ? w[r + 2] : w[r];
                const uint2 got = make_uint2(__shfl_xor(static_cast<int>(give.x), 4), __shfl_xor(static_cast<int>(give.y), 4));
                o[r] = hi ? u32x4{got.x, got.y, own.x, own.y} : u32x4{own.x, own.y, got.x, got.y};
            }
            if (8u * u >= g.width) return;
            u32x4* dst = reinterpret_cast<u32x4*>(g.k + codes + q8_k_off(j + (hi ? 2u : 0u), 8u * (u & ~4u), g.width));
            dst[0] = o[0];
            dst[1] = o[1];
            return;
        }
    }
    if (u >= cph) return;
#pragma unroll
    for (uint32_t r = 0; r < RB; r++) {
        if (!(R.held >> r & 1u)) continue;
        const uint32_t j = R.pos[r] & ((1u << g.page_shift) - 1u);
        const uint64_t pi = q8_page_index(g, R.h, R.page[r]);
        const uint64_t codes = (pi << g.page_shift) * g.width;
        if (!is_v) {
            *reinterpret_cast<uint2*>(g.k + codes + q8_k_off(j, 8u * u, g.width)) = w[r];
        } else {
            uint8_t* dst = g.v + codes + q8_v_off(j, 8u * u, g.width);
#pragma unroll
            for (int e = 0; e < 8; e++) dst[4 * e] = static_cast<uint8_t>((e < 4 ? w[r].x : w[r].y) >> (8 * (e & 3)));
        }
        if (u == 0) g.s[(pi << g.page_shift) * 2u + q8_s_off(j, is_v)] = static_cast<uint8_t>(b[r]);
    }
}

struct Q8LoadArgs {
    Q8Geom g;
    void* k_dst;  // [m, kv_heads, head_dim]
    void* v_dst;
    uint32_t k_wgs;
};

template <uint32_t DT, uint32_t RB>
__global__ __launch_bounds__(256) void q8_load_kernel(Q8LoadArgs a) {
    const Q8Geom& g = a.g;
    const bool is_v = blockIdx.x >= a.k_wgs;
    const Q8Rows<RB> R(g, is_v ? blockIdx.x - a.k_wgs : blockIdx.x);
    const uint32_t u = R.u;
    if (8u * u >= g.head_dim) return;
    uint2 w[RB];
    uint32_t b[RB];
    bool run = false;
    if constexpr (RB == 4) run = R.run && is_v;
    if (run) {  // the 4-slot words of V, transposed
        if constexpr (RB == 4) {
            const uint32_t j = R.pos[0] & ((1u << g.page_shift) - 1u);
            const uint64_t pi = q8_page_index(g, R.h, R.page[0]);
            const u32x4* src = reinterpret_cast<const u32x4*>(g.v + (pi << g.page_shift) * g.width + q8_v_off(j, 8u * u, g.width));
            const uint32_t sw = *reinterpret_cast<const uint32_t*>(g.s + (pi << g.page_shift) * 2u + q8_s_off(j, true));
            const u32x4 t[2] = {src[0], src[1]};
#pragma unroll
            for (int r = 0; r < 4; r++) b[r] = sw >> (8 * r) & 255u;
#pragma unroll
            for (int d = 0; d < 2; d++) {
                const uint32_t a01 = __builtin_amdgcn_perm(t[d][1], t[d][0], 0x05010400), b01 = __builtin_amdgcn_perm(t[d][1], t[d][0], 0x07030602);
                const uint32_t a23 = __builtin_amdgcn_perm(t[d][3], t[d][2], 0x05010400), b23 = __builtin_amdgcn_perm(t[d][3], t[d][2], 0x07030602);
                const uint32_t o[4] = {__builtin_amdgcn_perm(a23, a01, 0x05040100), __builtin_amdgcn_perm(a23, a01, 0x07060302),
                                       __builtin_amdgcn_perm(b23, b01, 0x05040100), __builtin_amdgcn_perm(b23, b01, 0x07060302)};
#pragma unroll
                for (int r = 0; r < 4; r++) (d ? w[r].y : w[r].x) = o[r];
            }
        }
    } else {
#pragma unroll
        for (uint32_t r = 0; r < RB; r++) {
            w[r] = make_uint2(0u, 0u);
            b[r] = 1u;
            if (!(R.held >> r & 1u)) continue;
            const uint32_t j = R.pos[r] & ((1u << g.page_shift) - 1u);
            const uint64_t pi = q8_page_index(g, R.h, R.page[r]);
            const uint64_t codes = (pi << g.page_shift) * g.width;
            b[r] = g.s[(pi << g.page_shift) * 2u + q8_s_off(j, is_v)];
            if (!is_v) {
                w[r] = *reinterpret_cast<const uint2*>(g.k + codes + q8_k_off(j, 8u * u, g.width));
            } else {
                const uint8_t* src = g.v + codes + q8_v_off(j, 8u * u, g.width);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    w[r].x |= static_cast<uint32_t>(src[4 * e]) << (8 * e);
                    w[r].y |= static_cast<uint32_t>(src[16 + 4 * e]) << (8 * e);
                }
            }
        }
    }
#pragma unroll
    for (uint32_t r = 0; r < RB; r++) {
        if (!(R.held >> r & 1u)) continue;
        float x[8];
        q8_decode8(w[r], __uint_as_float(b[r] << 23), x);
        q8_put8<DT>(is_v ? a.v_dst : a.k_dst,
                    (static_cast<uint64_t>(R.row0 + r) * g.kv_heads + R.h) * g.head_dim + 8u * u, x);
    }
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

// Rows a lane handles: 4 where the call still has two waves per SIMD, which
// fetch 4 rows each before they store the first.
uint32_t q8_rows_per_lane(const Q8Geom& g, uint32_t cus) {
    return (2ull * g.m * g.kv_heads << g.seg_shift) >= 64ull * 4 * 8 * cus ? 4u : 1u;
}

// Workgroups of one operand (K or V) of m rows, rb a lane.
uint32_t q8_wgs(const Q8Geom& g, uint32_t rb) {
    const uint64_t rows = rb > 1 ? static_cast<uint64_t>(g.m) + 2 * (rb - 1) : g.m;  // (groups are shifted by up to rb - 1)
    const uint64_t vecs = rows / rb * g.kv_heads, per = 4ull * (64u >> g.seg_shift);
    const uint64_t n = (vecs + per - 1) / per;
    if (static_cast<uint64_t>(g.m) * g.kv_heads > 0x7FFFFFFFull || n > 0x3FFFFFFFull)
        throw HipError{hipErrorInvalidConfiguration, "append grid too large"};
    return static_cast<uint32_t>(n);
}

template <uint32_t DT>
void store_rows(uint32_t rb, const Q8StoreArgs& a, hipStream_t s) {
    const dim3 grid(2 * a.k_wgs);
    if (rb == 4)
        hipLaunchKernelGGL((q8_store_kernel<DT, 4>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((q8_store_kernel<DT, 1>), grid, dim3(256), 0, s, a);
}

template <uint32_t DT>
void load_rows(uint32_t rb, const Q8LoadArgs& a, hipStream_t s) {
    const dim3 grid(2 * a.k_wgs);
    if (rb == 4)
        hipLaunchKernelGGL((q8_load_kernel<DT, 4>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((q8_load_kernel<DT, 1>), grid, dim3(256), 0, s, a);
}

}  // namespace

void launch_q8_store(thb_pool* p, uint32_t layer, const void* k_src, const void* v_src, uint32_t src_dtype,
                     const thb_rope* rope, const thb_rows* rows, uint32_t row_off, uint32_t m, hipStream_t s) {
    Q8StoreArgs a;
    a.g = q8_geom(p, layer, rows, row_off, m);
    const uint32_t rb = q8_rows_per_lane(a.g, p->cus);
    a.k_src = k_src;
    a.v_src = v_src;
    a.k_wgs = q8_wgs(a.g, rb);
    a.rope_on = rope != nullptr;
    a.rope = rope ? rope_dev(*rope, false) : RopeDev{};
    switch (src_dtype) {
        case THB_DT_F32: store_rows<THB_DT_F32>(rb, a, s); break;
        case THB_DT_F16: store_rows<THB_DT_F16>(rb, a, s); break;
        default: store_rows<THB_DT_BF16>(rb, a, s); break;
    }
    THB_HIP(hipGetLastError());
}

void launch_q8_load(thb_pool* p, uint32_t layer, void* k_dst, void* v_dst, uint32_t dst_dtype, const thb_rows* rows,
                    uint32_t row_off, uint32_t m, hipStream_t s) {
    Q8LoadArgs a;
    a.g = q8_geom(p, layer, rows, row_off, m);
    const uint32_t rb = q8_rows_per_lane(a.g, p->cus);
    a.k_dst = k_dst;
    a.v_dst = v_dst;
    a.k_wgs = q8_wgs(a.g, rb);
    switch (dst_dtype) {
        case THB_DT_F32: load_rows<THB_DT_F32>(rb, a, s); break;
        case THB_DT_F16: load_rows<THB_DT_F16>(rb, a, s); break;
        default: load_rows<THB_DT_BF16>(rb, a, s); break;
    }
    THB_HIP(hipGetLastError());
}

}  // namespace thb
