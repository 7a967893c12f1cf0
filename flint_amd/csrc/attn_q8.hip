// Paged attention over an 8-bit pool (THB_KV_E4M3; format and page layout in
// q8.hpp), on the work items, row ranges and partial results of attention.hip.
//
// Mathematics.  With code vectors c and scales 2^e of a head's keys and values,
//   s_j = 2^ek_j (q . ck_j) scale,   y = sum_j p_j 2^ev_j cv_j / sum_j p_j,
// p_j = exp(s_j - max).  The scales are powers of two, one per token, so they
// stay out of the products: the key's multiplies its score, the value's its
// probability (both exact), and the matrix cores see the codes, which are exact
// in f16 and bf16 (4 significant bits).
//  * QK^T in f16: the query vector is scaled by a power of two to a largest
//    element in [2^14, 2^15) (exact; undone in the f32 scores), where an f16 or
//    bf16 query is one exact f16 operand and an f32 or rotated one is split into
//    a high and a low half (22 bits).
//  * PV in bf16, whose exponents hold p_j 2^ev_j for any scale; the product is
//    split into a high and a low half (16 bits, 2^-17 of each term).  The sum of
//    the probabilities is kept in f32 from the unrounded ones.
#include "attn_decode.hpp"
#include "q8.hpp"

namespace thb {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// 8 codes (two words) as f16.
__device__ __forceinline__ f16x8 q8_f16(uint32_t w0, uint32_t w1) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The same as bf16.
__device__ __forceinline__ bf16x8 q8_bf16(uint32_t w0, uint32_t w1) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// Scale of byte e (0 .. 3) of a word: 255 gives an infinity, which makes the
// zero codes beside it NaN.
__device__ __forceinline__ float q8_scale(uint32_t w, int e) {
    const uint32_t b = e == 0 ? w << 23 : e == 1 ? w << 15 : e == 2 ? w << 7 : w >> 1;
    return __uint_as_float(b & 0x7f800000u);
}
// High and low bf16 parts of 8 values.
__device__ __forceinline__ void split_bf16(const float (&x)[8], bf16x8& h, bf16x8& l) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const bf16x2 hh = __builtin_convertvector((f32x2{x[e], x[e + 1]}), bf16x2);
        const bf16x2 ll = __builtin_convertvector(
            (f32x2{x[e] - static_cast<float>(hh[0]), x[e + 1] - static_cast<float>(hh[1])}), bf16x2);
        h[e] = hh[0];
        h[e + 1] = hh[1];
        l[e] = ll[0];
        l[e + 1] = ll[1];
    }
}

// The query operand of a lane (load_q_f32's elements) in f16, scaled by a power
// of two; returns the factor that undoes the scaling.  Every lane must call it.
template <int KS, bool QLO, bool FULL>
__device__ __forceinline__ float load_q_scaled(const AttnArgs& a, bool con, uint32_t row, uint32_t head, uint32_t a4,
                                               f16x8 (&qh)[KS], f16x8 (&ql)[QLO ? KS : 1]) {
    uint32_t ef = 15u;
    load_q_f32<KS, FULL>(a, con, row, head, a4, [&](float (&x)[KS][8]) {
        uint32_t mx = 0u;
#pragma unroll
        for (int j = 0; j < KS; j++) mx = max(mx, q8_amax8(x[j]));
        mx = max(mx, static_cast<uint32_t>(__shfl_xor(static_cast<int>(mx), 16)));
        mx = max(mx, static_cast<uint32_t>(__shfl_xor(static_cast<int>(mx), 32)));
        ef = min(max(mx >> 23, 15u), 253u);
        const float down = __uint_as_float((268u - ef) << 23);
#pragma unroll
        for (int j = 0; j < KS; j++) {
#pragma unroll
            for (int e = 0; e < 8; e++) x[j][e] *= down;
            if constexpr (QLO) {
                Ops<true>::split8_fast(x[j], qh[j], ql[j]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) qh[j][e] = static_cast<_Float16>(x[j][e]);
            }
        }
    });
    return __uint_as_float((ef - 14u) << 23);
}

constexpr int q8_waves(int hd) { return hd >= 512 ? 4 : 8; }
constexpr int q8_ring(int hd) { return hd <= 64 ? 4 : hd <= 128 ? 2 : 1; }

template <int HD, int W>
struct Q8Lds {
    uint32_t page[kMaxPartPages];
    f32x4 o[W][HD / 16][64];
    float m[W][64];
    float l[W][64];
    uint32_t arrived;  // partitions of the group finished before this one
};

// One (group, partition, KV head) per workgroup of W waves, which split the
// partition's keys into W runs of 32-key steps and keep NB steps in flight each.
template <int HD, int W, int NB, bool QLO, bool FULL>
__global__ __launch_bounds__(64 * W) void attn_q8(AttnArgs a) {
    constexpr int KS = HD / 32;  // QK k-steps of 32 dimensions
    constexpr int KB = HD / 64;  // 1 KiB blocks of a 16-key tile
    constexpr int MT = HD / 16;  // PV tiles
    __shared__ Q8Lds<HD, W> L;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t a4 = lane >> 4, c = lane & 15u;
    const uint32_t item = blockIdx.x / a.n_kvh, kvh = blockIdx.x - item * a.n_kvh;
    const uint32_t* G = a.items + static_cast<uint64_t>(item) * kItemWords;
    const uint32_t r0 = G[0], R = G[1], h0 = G[2], H = G[3], seq = G[4];
    const uint32_t glo = G[5], ghi = G[6], n_parts = G[7], gbase = G[8], P = G[9], item0 = G[10];
    const uint32_t part = G[kGroupWords], part_slot = item0 + part;
    if (part >= n_parts) return;  // a device plan's unused slot
    const uint32_t pbeg = gbase + part * P;
    const uint32_t tb = max(glo, pbeg), te = min(ghi, pbeg + P);
    const uint32_t hd = a.head_dim, width = q8_width(hd);
    const uint32_t pshift = a.page_shift, pmask = (1u << pshift) - 1u;

    // This wave's run of keys [ws, we).
    const uint32_t tb16 = tb & ~15u;
    const uint32_t span = te > tb16 ? te - tb16 : 0u;
    const uint32_t run = ((span + W - 1) / W + 31u) & ~31u;
    const uint32_t ws = tb16 + wave * run, we = min(ws + run, te);

    const uint32_t lp0 = pbeg >> pshift;
    {
        const uint32_t npg = P >> pshift;
        const uint32_t* trow = a.table + static_cast<uint64_t>(seq) * a.max_pages;
        for (uint32_t i = tid; i < npg; i += 64 * W) {
            const uint32_t lp = lp0 + i;
            const bool used = tb < te && (lp << pshift) < te && ((lp + 1) << pshift) > tb;
            const uint32_t pg = used ? trow[lp] : 0u;
            L.page[i] = pg < a.pages ? pg : 0u;  // block_pages: a page outside the pool reads page 0
        }
    }

    // Column c of this lane: row r0 + c / H, head h0 + c % H of the KV head.
    const uint32_t ncols = R * H;
    const bool con = c < ncols;
    const uint32_t rr = con ? c / H : 0u;
    const uint32_t row = r0 + rr;
    const uint32_t head = kvh * a.nq_per_kv + h0 + (con ? c - rr * H : 0u);
    uint32_t clo = 0, chi = 0;
    if (con) {
        clo = max(a.ranges[2 * row], tb);
        chi = min(a.ranges[2 * row + 1], we);
    }
    const uint32_t cspan = chi > clo ? chi - clo : 0u;  // key t is read iff t - clo < cspan

    f16x8 qh[KS], ql[QLO ? KS : 1];
    const float qf = load_q_scaled<KS, QLO, FULL>(a, con, row, head, a4, qh, ql) * a.qscale;
    __syncthreads();

    float m = kFloor, l = 0.0f;
    f32x4 o[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // A step's operands: two 16-key tiles.  Tiles past the run repeat its last
    // one (their keys are masked), blocks past the row width its first (the
    // query is zero there, and such outputs are never stored): every step issues
    // the same loads, all inside the pool.
    struct Step {
        u32x4 k[2][KB], v[2][KB];
        u32x2 s[2];
    };
    const uint32_t last = we > ws ? (we - 1u) & ~15u : 0u;
    const uint32_t nb = width >> 6;
    const uint8_t* kcodes = reinterpret_cast<const uint8_t*>(a.k);
    const uint8_t* vcodes = reinterpret_cast<const uint8_t*>(a.v);
    auto load = [&](uint32_t t0, Step& x) {
#pragma unroll
        for (uint32_t u = 0; u < 2; u++) {
            const uint32_t t = min(t0 + 16u * u, last);
            const uint32_t page = __builtin_amdgcn_readfirstlane(L.page[(t >> pshift) - lp0]);
            const uint64_t slot = ((static_cast<uint64_t>(kvh) * a.pages + page) << pshift) + (t & pmask);
            const uint8_t* kp = kcodes + slot * width;
            const uint8_t* vp = vcodes + slot * width;
            x.s[u] = *reinterpret_cast<const u32x2*>(a.scales + slot * 2u + 8u * a4);
#pragma unroll
            for (uint32_t j = 0; j < KB; j++) {
                const uint32_t at = (j < nb ? j << 10 : 0u) + 16u * lane;
                x.k[u][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + at));
            }
#pragma unroll
            for (uint32_t j = 0; j < KB; j++) {
                const uint32_t at = (j < nb ? j << 10 : 0u) + 16u * lane;
                x.v[u][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vp + at));
            }
        }
    };
    const float cap2 = a.cap2;
    auto compute = [&](uint32_t t0, const Step& x) {
        f32x4 s[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int j = 0; j < KS; j++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const f16x8 kc = q8_f16(x.k[u][j >> 1][2 * (j & 1)], x.k[u][j >> 1][2 * (j & 1) + 1]);
                s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, qh[j], s[u], 0, 0, 0);
                if constexpr (QLO) s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, ql[j], s[u], 0, 0, 0);
            }
        float sv[8], mx = -INFINITY;
        bool in[8];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float y = s[u][e] * (q8_scale(x.s[u][0], e) * qf);
                if (FULL && cap2 != 0.0f) y = cap2 * tanh_approx(y);
                const uint32_t t = t0 + 16u * u + 4u * a4 + e;
                in[4 * u + e] = t - clo < cspan;
                y = in[4 * u + e] ? y : -INFINITY;
                sv[4 * u + e] = y;
                mx = fmaxf(mx, y);
            }
        // Lazy rescale: the running max moves only when a score beats it by
        // more than kTau.
        if (__builtin_amdgcn_ballot_w64(mx > m + kTau) != 0) {
            mx = col_max(mx);
            if (mx > m + kTau) {
                const float alpha = fast_exp2(m - mx);
                l *= alpha;
#pragma unroll
                for (int i = 0; i < MT; i++) o[i] *= alpha;
                m = mx;
            }
        }
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float pe = fast_exp2(sv[e] - m);
            l += pe;
            // (A masked slot's scale may be anything.)
            p[e] = in[e] ? pe * q8_scale(x.s[e >> 2][1], e & 3) : 0.0f;
        }
        bf16x8 ph, pl;
        split_bf16(p, ph, pl);
#pragma unroll
        for (int j = 0; j < KB; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bf16x8 vc = q8_bf16(x.v[0][j][i], x.v[1][j][i]);
                o[4 * j + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vc, ph, o[4 * j + i], 0, 0, 0);
                o[4 * j + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vc, pl, o[4 * j + i], 0, 0, 0);
            }
    };

    if (ws < we) {
        Step x[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) load(ws + 32u * b, x[b]);
        for (uint32_t t0 = ws; t0 < we; t0 += 32u * NB) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint32_t t = t0 + 32u * b;
                if (t < we) compute(t, x[b]);
                load(t + 32u * NB, x[b]);
            }
        }
    }
    l = col_sum(l);

    // Merge the waves' states.  Element e of output tile 4 j + i is dim 64 j +
    // 16 a4 + 4 e + i: unit 4 j + e holds 4 consecutive dims.
#pragma unroll
    for (int j = 0; j < KB; j++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            L.o[wave][4 * j + e][lane] = f32x4{o[4 * j][e], o[4 * j + 1][e], o[4 * j + 2][e], o[4 * j + 3][e]};
    L.m[wave][lane] = m;
    L.l[wave][lane] = l;
    __syncthreads();
    float wm[W], wl[W], f[W], M, Ls;
#pragma unroll
    for (int w = 0; w < W; w++) {
        wm[w] = L.m[w][lane];
        wl[w] = L.l[w][lane];
    }
    wave_weights<W>(wm, wl, f, M, Ls);
    const uint64_t pb = (static_cast<uint64_t>(part_slot) * a.n_kvh + kvh) * kCols + c;
    for (uint32_t i = wave; i < static_cast<uint32_t>(MT); i += W) {
        f32x4 acc = L.o[0][i][lane] * f[0];
#pragma unroll
        for (int w = 1; w < W; w++) acc = fma4(L.o[w][i][lane], f[w], acc);
        const uint32_t d = 64u * (i >> 2) + 16u * a4 + 4u * (i & 3u);
        if (!con || d >= hd) continue;
        if (n_parts == 1) {
            const f32x4 yv = acc * (1.0f / Ls);
            const float v4[4] = {yv[0], yv[1], yv[2], yv[3]};
            store_y<4, FULL>(a, row, head, d, v4);
        } else {
            publish_o(a.part_o + pb * HD + d, acc);
        }
    }
    if (n_parts > 1 && wave == 0 && con && a4 == 0) publish_ml(a.part_ml + 2 * pb, M, Ls);
    if (n_parts > 1 && a.merge_cnt)
        merge_if_last<HD, FULL, 64 * W>(a, L.arrived, r0, R, h0, H, n_parts, item0, kvh, tid);
}

// An f16 or bf16 query read as it is needs no low half.
bool q8_query_lo(const AttnArgs& a) { return a.q_dt == THB_DT_F32 || a.rope_on; }

template <int HD>
void launch_q8_hd(dim3 grid, const AttnArgs& a, hipStream_t s) {
    constexpr int W = q8_waves(HD), NB = q8_ring(HD);
    const bool lo = q8_query_lo(a);
    if (a.full && lo)
        hipLaunchKernelGGL((attn_q8<HD, W, NB, true, true>), grid, dim3(64 * W), 0, s, a);
    else if (a.full)
        hipLaunchKernelGGL((attn_q8<HD, W, NB, false, true>), grid, dim3(64 * W), 0, s, a);
    else if (lo)
        hipLaunchKernelGGL((attn_q8<HD, W, NB, true, false>), grid, dim3(64 * W), 0, s, a);
    else
        hipLaunchKernelGGL((attn_q8<HD, W, NB, false, false>), grid, dim3(64 * W), 0, s, a);
}

}  // namespace

void launch_q8_decode(uint32_t hd, dim3 grid, const AttnArgs& a, hipStream_t s) {
    switch (hd) {
        case 64: launch_q8_hd<64>(grid, a, s); break;
        case 128: launch_q8_hd<128>(grid, a, s); break;
        case 256: launch_q8_hd<256>(grid, a, s); break;
        default: launch_q8_hd<512>(grid, a, s); break;
    }
}

}  // namespace thb
