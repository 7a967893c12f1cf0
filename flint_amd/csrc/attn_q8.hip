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
//    split into a high and a low part (16 bits, 2^-17 of each term) for a 16-bit
//    output and a third (24 bits) for f32 (two leave 2e-6 to 3.4e-6 of an output's
//    size, three under 1e-6; 1000 rows after 3000 keys at head_dim 256 159 / 170
//    us, decode unchanged).  The sum of the probabilities is kept
//    in f32 from the unrounded ones.
#include <type_traits>

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
// N bf16 parts of 8 values, the highest first.
template <int N>
__device__ __forceinline__ void split_bf16(float (&x)[8], bf16x8 (&part)[N]) {
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const bf16x2 hh = __builtin_convertvector((f32x2{x[e], x[e + 1]}), bf16x2);
            part[n][e] = hh[0];
            part[n][e + 1] = hh[1];
            x[e] -= static_cast<float>(hh[0]);
            x[e + 1] -= static_cast<float>(hh[1]);
        }
}

// Soft-capped scores, cap2 * tanh(y).  They are mostly small beside the cap, where
// 1 - 2 / (exp(2y) + 1) would leave 2^-23 of the whole cap: below 1/4 the odd
// Taylor polynomial (the next term is 2^-26 of y), and (1 - t) / (1 + t) of t =
// exp(-2|y|) where some score of the wave is above.
__device__ __forceinline__ void soft_cap(float (&y)[8], float cap2) {
    float r[8];
    bool big = false;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float y2 = y[e] * y[e];
        float t = __builtin_fmaf(y2, 62.0f / 2835.0f, -17.0f / 315.0f);
        t = __builtin_fmaf(t, y2, 2.0f / 15.0f);
        t = __builtin_fmaf(t, y2, -1.0f / 3.0f);
        r[e] = __builtin_fmaf(t * y2, y[e], y[e]);
        big = big || !(y2 < 0.0625f);
    }
    if (__builtin_amdgcn_ballot_w64(big) != 0) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float t = fast_exp2(__builtin_fabsf(y[e]) * -2.8853900817779268f);  // -2 log2(e)
            const float z = __builtin_copysignf((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t), y[e]);
            r[e] = y[e] * y[e] < 0.0625f ? r[e] : z;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = cap2 * r[e];
}

// The query operand of a lane (load_q_f32's elements) in f16, scaled by a power
// of two and by pre (1 or -1); returns the factor that undoes the power of two.
// Every lane must call it.
template <int KS, bool QLO, bool FULL>
__device__ __forceinline__ float load_q_scaled(const AttnArgs& a, bool con, uint32_t row, uint32_t head, uint32_t a4,
                                               f16x8 (&qh)[KS], f16x8 (&ql)[QLO ? KS : 1], float pre = 1.0f) {
    uint32_t ef = 15u;
    load_q_f32<KS, FULL>(a, con, row, head, a4, [&](float (&x)[KS][8]) {
        uint32_t mx = 0u;
#pragma unroll
        for (int j = 0; j < KS; j++) mx = max(mx, q8_amax8(x[j]));
        mx = max(mx, static_cast<uint32_t>(__shfl_xor(static_cast<int>(mx), 16)));
        mx = max(mx, static_cast<uint32_t>(__shfl_xor(static_cast<int>(mx), 32)));
        ef = min(max(mx >> 23, 15u), 253u);
        const float down = __uint_as_float((268u - ef) << 23) * pre;
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
// PP: bf16 parts of the probabilities.
template <int HD, int W, int NB, bool QLO, int PP, bool FULL>
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
            for (int e = 0; e < 4; e++) sv[4 * u + e] = s[u][e] * (q8_scale(x.s[u][0], e) * qf);
        if (FULL && cap2 != 0.0f) soft_cap(sv, cap2);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t t = t0 + 16u * (e >> 2) + 4u * a4 + (e & 3);
            in[e] = t - clo < cspan;
            sv[e] = in[e] ? sv[e] : -INFINITY;
            mx = fmaxf(mx, sv[e]);
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
        bf16x8 part[PP];
        split_bf16<PP>(p, part);
#pragma unroll
        for (int j = 0; j < KB; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bf16x8 vc = q8_bf16(x.v[0][j][i], x.v[1][j][i]);
#pragma unroll
                for (int n = 0; n < PP; n++)
                    o[4 * j + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vc, part[n], o[4 * j + i], 0, 0, 0);
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

// ---------------------------------------------------------------- chunks
// Prefill blocks: many query vectors read the same keys, so the codes are
// converted once per call (q8_expand) into f16 in the order the matrix cores take
// them, which the attention kernel then moves to LDS without touching a register.
// (Converted by every workgroup on its way to LDS, the codes cost as many vector
// instructions as the softmax: 251 us for the 4096-token prompt.)
//
// Scales.  Per step of 32 keys, K's and V's largest scales are taken out as a
// reference: codes become code * 2^(e - ref + 7) in f16 (at most 57344; exact
// down to e = ref - 22, below that off by at most 2^-25 of a step whose largest
// value is 2^15.8).  K's reference goes into the factor of the step's scores.
// V's reference less the accumulators' own (an exponent, raised rarely, with
// all the accumulators, when a step's is above it) goes into the exponent of the
// probabilities.  So a score costs no multiply for either scale.  Probabilities
// are 2^kPBias times too large throughout, which keeps them clear of f16's
// subnormals (at most 2^(kPBias + kTau) = 2^15), and are one f16 operand for a
// 16-bit output (each off by at most 2^-11 of itself, an f16 output's own rounding) or split into
// two for f32 (PLO).  The sum l is taken from the unrounded ones.
//
// Bound by the matrix cores and the exponentials: the 4096-token prompt of 8 KV
// heads of 128 x 4 takes 182 us in all, 11 of them the expansion: 752 TFLOP/s.
constexpr float kPBias = 7.0f;
constexpr uint32_t kQ8Up = 7;

// One step's references: K's, V's (bit 31: the step holds NaN values), and the
// NaN values among each lane group's 8 keys, a bit each.
struct Q8Ref {
    uint32_t k, v, pad[2], nan[4];
};
static_assert(sizeof(Q8Ref) == kQ8RefBytes, "scratch layout");

// 2^n for an exponent field, 0 below the normal range.
__device__ __forceinline__ float pow2_field(int32_t field) {
    return __uint_as_float(field > 0 ? static_cast<uint32_t>(field) << 23 : 0u);
}
// Maximum over the 16 lanes of a lane group (DPP row rotations) / over the 4
// lane groups, each of which holds one value.
template <int CTRL>
__device__ __forceinline__ uint32_t row_perm(uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t max16(uint32_t x) {
    x = max(x, row_perm<0x128>(x));
    x = max(x, row_perm<0x124>(x));
    x = max(x, row_perm<0x122>(x));
    return max(x, row_perm<0x121>(x));
}
__device__ __forceinline__ uint32_t max_groups(uint32_t x) {
    const uint32_t g0 = __builtin_amdgcn_readlane(x, 0), g1 = __builtin_amdgcn_readlane(x, 16);
    const uint32_t g2 = __builtin_amdgcn_readlane(x, 32), g3 = __builtin_amdgcn_readlane(x, 48);
    return max(max(g0, g1), max(g2, g3));
}

// Expands the keys of a call's prefill blocks: workgroup (step, KV head), its
// waves the 64-dim blocks of K and of V.  Scratch per KV head: HD / 8 units per
// step, K [16-key tile][k-step] then V [output tile], 1 KiB each; and a Q8Ref a
// step.  Keys outside a region's [lo, hi) are clamped to its first or last 16.
template <int HD>
__global__ __launch_bounds__(64 * (HD / 64) * 2) void q8_expand(AttnArgs a) {
    constexpr uint32_t KB = HD / 64, KS = HD / 32;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t a4 = lane >> 4, c = lane & 15u, kvh = blockIdx.y;
    // The step's region: the last that starts at or before it.
    uint32_t before = 0;
    for (uint32_t r = lane; __builtin_amdgcn_ballot_w64(r < a.n_regions) != 0; r += 64u)
        before += __builtin_popcountll(
            __builtin_amdgcn_ballot_w64(r < a.n_regions && a.regions[r * kQ8RegionWords + 3] <= blockIdx.x));
    const uint32_t* R = a.regions + (before - 1u) * kQ8RegionWords;
    const uint32_t lo = R[1], hi = R[2];
    const uint32_t t0 = ((lo >> 5) + (blockIdx.x - R[3])) << 5;
    const uint32_t first16 = lo & ~15u, last16 = (hi - 1u) & ~15u;
    const uint32_t hd = a.head_dim, width = q8_width(hd), nb = width >> 6;
    const uint32_t pshift = a.page_shift, pmask = (1u << pshift) - 1u;
    const uint32_t* trow = a.table + static_cast<uint64_t>(R[0]) * a.max_pages;
    const bool is_v = wave >= KB;
    const uint32_t j = wave - (is_v ? KB : 0u);
    const uint8_t* codes = reinterpret_cast<const uint8_t*>(is_v ? a.v : a.k);
    u32x4 cw[2];
    uint32_t sw[2];
#pragma unroll
    for (uint32_t h = 0; h < 2; h++) {
        const uint32_t t = min(max(t0 + 16u * h, first16), last16);
        uint32_t page = trow[t >> pshift];
        page = page < a.pages ? page : 0u;  // block_pages: a page outside the pool reads page 0
        const uint64_t slot = ((static_cast<uint64_t>(kvh) * a.pages + page) << pshift) + (t & pmask);
        cw[h] = *reinterpret_cast<const u32x4*>(codes + slot * width + (j < nb ? j << 10 : 0u) + 16u * lane);
        const uint8_t* sc = a.scales + slot * 2u;
        sw[h] = is_v ? *reinterpret_cast<const uint32_t*>(sc + 8u * a4 + 4u) : sc[(c >> 2) * 8u + (c & 3u)];
        // Keys that no row reads (whatever their slots hold) have no say in the references.
        const uint32_t u = t0 + 16u * h + (is_v ? 4u * a4 : c);
        if (is_v) {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) sw[h] &= u + e - lo < hi - lo ? ~0u : ~(255u << (8u * e));
        } else {
            sw[h] = u - lo < hi - lo ? sw[h] : 0u;
        }
    }
    const uint64_t at = static_cast<uint64_t>(kvh) * a.steps + blockIdx.x;
    u32x4* base = reinterpret_cast<u32x4*>(a.expanded);
    u32x4* dst = base + at * (KS * 4u * 64u) + lane;
    Q8Ref* ref_at = reinterpret_cast<Q8Ref*>(base + static_cast<uint64_t>(a.n_kvh) * a.steps * (KS * 4u * 64u)) + at;
    if (!is_v) {
        const uint32_t ref = max(max16(max(sw[0] == 255u ? 0u : sw[0], sw[1] == 255u ? 0u : sw[1])), kQ8Up + 1u);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float f = pow2_field(127 + static_cast<int32_t>(kQ8Up) + static_cast<int32_t>(sw[h]) -
                                       static_cast<int32_t>(ref));
#pragma unroll
            for (int q = 0; q < 2; q++) {
                u32x4 w;
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    const uint32_t x = cw[h][2 * q + d];
                    w[2 * d] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, f, false));
                    w[2 * d + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, f, true));
                }
                if (sw[h] == 255u) w = u32x4{0x7E007E00u, 0x7E007E00u, 0x7E007E00u, 0x7E007E00u};  // a NaN key
                dst[(h * KS + 2 * j + q) * 64u] = w;
            }
        }
        if (j == 0 && lane == 0) ref_at->k = ref;
        return;
    }
    uint32_t ref = 0u, nan = 0u, bb[2][4];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t b = (sw[h] >> (8 * e)) & 255u;
            bb[h][e] = b == 255u ? 0u : b;
            nan |= b == 255u ? 1u << (4 * h + e) : 0u;
            ref = max(ref, bb[h][e]);
        }
    ref = max(max_groups(ref), kQ8Up + 1u);
    f16x2 f[2][2];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            f[h][e >> 1][e & 1] = static_cast<_Float16>(pow2_field(
                127 + static_cast<int32_t>(kQ8Up) + static_cast<int32_t>(bb[h][e]) - static_cast<int32_t>(ref)));
#pragma unroll
    for (int d = 0; d < 4; d++) {
        u32x4 w;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const f16x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(cw[h][d], 1.0f, false);
            const f16x2 v1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(cw[h][d], 1.0f, true);
            w[2 * h] = __builtin_bit_cast(uint32_t, v0 * f[h][0]);
            w[2 * h + 1] = __builtin_bit_cast(uint32_t, v1 * f[h][1]);
        }
        dst[(2u * KS + 4u * j + d) * 64u] = w;
    }
    if (j == 0) {
        const bool any = __builtin_amdgcn_ballot_w64(nan != 0u) != 0;
        if (c == 0) ref_at->nan[a4] = nan;
        if (lane == 0) ref_at->v = ref | (any ? 1u << 31 : 0u);
    }
}

template <int HD>
struct Q8PrefillLds {
    union {
        struct {
            u32x4 k[3][2][HD / 32][64];  // [32-key step % 3][16-key tile][k-step]
            u32x4 v[3][HD / 16][64];     // [32-key step % 3][output tile]
        };
        u32x4 out[kQ8PrefillWaves][4][64];  // behind the steps: the waves' outputs, 64 dims at a time
    };
};

// Schedules a block of N LDS operand reads, each feeding M products: kAhead
// reads, then products and reads in turn (left to itself the compiler waits for
// every other read, or keeps so many in registers that others spill).
template <int N, int M>
__device__ __forceinline__ void order_reads() {
    constexpr int kAhead = 3;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);  // LDS reads
#pragma unroll
    for (int i = 0; i < N; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, M, 0);  // matrix products
        if (i + kAhead < N) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
}

// One workgroup of W = 4 waves handles a block of query groups for one KV head and
// one partition of the block's keys; wave w takes groups w and w + 4, up to NCG of
// them (16 query vectors each).  Per step of 32 keys a wave runs QK^T of the next
// step, the softmax of this one and PV; the matrix products of one workgroup go
// beside the softmax of another on the same CU: three at head_dim 128 (48 KiB of
// LDS and 168 registers each), or two with two groups a wave, which read each
// operand from LDS for twice the products.  (One workgroup of 8 waves with two
// groups each, in step at its barriers: 217 us for the 4096-token prompt, 191
// as two of 4; with the softmax's instructions between the products of the same
// wave 240.)
template <int HD, int NCG, bool QLO, bool PLO, bool CAP>
__global__ __launch_bounds__(64 * kQ8PrefillWaves, NCG == 2 ? 2 : HD <= 64 ? 4 : 3) void attn_q8_prefill(AttnArgs a) {
    constexpr uint32_t W = kQ8PrefillWaves;
    constexpr int KS = HD / 32, KB = HD / 64, MT = HD / 16;
    constexpr uint32_t UNITS = 2 * KS + MT;  // 1 KiB units of a step
    __shared__ Q8PrefillLds<HD> L;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t a4 = lane >> 4, c = lane & 15u;
    const uint32_t item = blockIdx.x / a.n_kvh, kvh = blockIdx.x - item * a.n_kvh;
    const uint32_t* B = a.bitems + static_cast<uint64_t>(item) * kBItemWords;
    const uint32_t g0 = B[0], ng = B[1], part = B[kBlockWords];
    const uint32_t n_parts = B[5], P = B[7], pbeg = B[6] + part * P;
    const BlockKeys keys = block_keys(B[3], B[4], pbeg, P, 32);
    const uint32_t tb = keys.tb, te = keys.te, S = keys.tiles;  // S steps of 32 keys
    const uint32_t hd = a.head_dim;
    // This block's steps in the scratch: slot of key 0's step (modulo 2^32) plus its own.
    const uint64_t step0 = static_cast<uint64_t>(kvh) * a.steps + (a.bregions[item] + (keys.first >> 5));
    const u32x4* base = reinterpret_cast<const u32x4*>(a.expanded);
    const u32x4* src = base + step0 * (UNITS * 64u);
    const Q8Ref* refs = reinterpret_cast<const Q8Ref*>(base + static_cast<uint64_t>(a.n_kvh) * a.steps * (UNITS * 64u)) + step0;

    // A step's units to LDS, spread over the waves.  (Past the last step it again:
    // unread.)
    const uint32_t k0 = __builtin_amdgcn_readfirstlane(lds_offset(&L.k[0][0][0][0]));
    const uint32_t v0 = __builtin_amdgcn_readfirstlane(lds_offset(&L.v[0][0][0]));
    auto request = [&](uint32_t n) __attribute__((always_inline)) {
        const u32x4* from = src + static_cast<uint64_t>(min(n, S - 1u)) * (UNITS * 64u);
#pragma unroll
        for (uint32_t i = 0; i < UNITS / W; i++) {
            const uint32_t u = wave + W * i;
            const uint32_t to = u < 2u * KS ? k0 + ((n % 3u) * 2u * KS + u) * 1024u
                                            : v0 + ((n % 3u) * MT + u - 2u * KS) * 1024u;
            dma16_from(from + u * 64u, 16u * lane, to);
        }
    };
    if (S) {
        request(0);
        request(1);
    }

    // Column c of this wave's g-th group, whose first partial-result slot it returns.
    auto column = [&](uint32_t g, bool& on, uint32_t& row, uint32_t& head) {
        const uint32_t gi = wave + W * g;
        const uint32_t* G = a.groups + (g0 + (gi < ng ? gi : 0u)) * kGroupWords;
        const uint32_t r0 = G[0], R = G[1], h0 = G[2], H = G[3];
        on = gi < ng && c < R * H;
        const uint32_t rr = on ? c / H : 0u;
        row = r0 + rr;
        head = kvh * a.nq_per_kv + h0 + (on ? c - rr * H : 0u);
        return G[10];
    };
    // This wave's groups and columns.
    bool con[NCG];
    uint32_t clo[NCG], cspan[NCG], lomax[NCG], himin[NCG];
    f16x8 qh[NCG][KS], ql[NCG][QLO ? KS : 1];
    float qf[NCG];
#pragma unroll
    for (int g = 0; g < NCG; g++) {
        uint32_t row, head;
        column(g, con[g], row, head);
        const uint32_t lo = con[g] ? max(a.ranges[2 * row], tb) : 0u;
        const uint32_t hi = con[g] ? min(a.ranges[2 * row + 1], te) : 0u;
        clo[g] = lo;
        cspan[g] = hi > lo ? hi - lo : 0u;  // key t is read iff t - clo < cspan
        // Steps inside [lomax, himin) of every column need no mask.
        uint32_t l2 = con[g] ? lo : 0u, h2 = con[g] ? hi : 0xFFFFFFFFu;
#pragma unroll
        for (int sh = 1; sh < 64; sh <<= 1) {
            l2 = max(l2, static_cast<uint32_t>(__shfl_xor(static_cast<int>(l2), sh)));
            h2 = min(h2, static_cast<uint32_t>(__shfl_xor(static_cast<int>(h2), sh)));
        }
        lomax[g] = __builtin_amdgcn_readfirstlane(l2);
        himin[g] = __builtin_amdgcn_readfirstlane(h2);
        // The sign of the score scale goes into the query, its size into qf >= 0.
        const float undo = load_q_scaled<KS, QLO, true>(a, con[g], row, head, a4, qh[g], ql[g], a.qpre);
        qf[g] = undo * a.qpost;
    }

    float m[NCG], l[NCG];
    f32x4 o[NCG][MT];
    int32_t oref = 0;  // the accumulators hold sums of value * 2^-(oref - 127)
#pragma unroll
    for (int g = 0; g < NCG; g++) {
        m[g] = kFloor;
        l[g] = 0.0f;
#pragma unroll
        for (int i = 0; i < MT; i++) o[g][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const float cap2 = a.cap2;
    // Scores of one step (16 keys each, soft-capped and masked), their factor (above 0:
    // a masked score stays -inf) and maxima; probabilities of one.
    typedef f32x4 Scores[NCG][2];
    Scores sc0, sc1;
    float kf[NCG], mx[NCG], alpha[NCG];
    f16x8 ph[NCG], pl[PLO ? NCG : 1];
    auto qk = [&](uint32_t n, Scores& sc) __attribute__((always_inline)) {  // of step n
#pragma unroll
        for (int g = 0; g < NCG; g++) sc[g][0] = sc[g][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < KS; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const f16x8 kc = __builtin_bit_cast(f16x8, L.k[n % 3u][h][j][lane]);
#pragma unroll
                for (int g = 0; g < NCG; g++) sc[g][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, qh[g][j], sc[g][h], 0, 0, 0);
                if constexpr (QLO) {
#pragma unroll
                    for (int g = 0; g < NCG; g++)
                        sc[g][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, ql[g][j], sc[g][h], 0, 0, 0);
                }
            }
    };
    // PV of step n; scaled: onto the accumulators times alpha.
    auto pv = [&](auto scaled_t, uint32_t n) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MT; i++) {
            const f16x8 vc = __builtin_bit_cast(f16x8, L.v[n % 3u][i][lane]);
#pragma unroll
            for (int g = 0; g < NCG; g++) {
                f32x4 acc = o[g][i];
                if constexpr (decltype(scaled_t)::value) acc *= alpha[g];
                o[g][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, ph[g], acc, 0, 0, 0);
            }
            if constexpr (PLO) {
#pragma unroll
                for (int g = 0; g < NCG; g++) o[g][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, pl[g], o[g][i], 0, 0, 0);
            }
        }
    };
    // Soft-cap, mask (masked_t) and maxima of the scores of 32 keys from ts.
    auto maxima = [&](auto masked_t, uint32_t ts, Scores& sc, float kscale) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < NCG; g++) {
            kf[g] = fmaxf(qf[g] * kscale, 1.17549435e-38f);
            if constexpr (CAP) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = sc[g][e >> 2][e & 3] * kf[g];
                soft_cap(y, cap2);
#pragma unroll
                for (int e = 0; e < 8; e++) sc[g][e >> 2][e & 3] = y[e];
            }
            if constexpr (decltype(masked_t)::value) {
                uint32_t t = ts + 4u * a4 - clo[g];
                asm volatile("" : "+v"(t));  // (else 8 sums a group are kept in registers through the loop)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    sc[g][e >> 2][e & 3] = t + (16u * (e >> 2) + (e & 3)) < cspan[g] ? sc[g][e >> 2][e & 3] : -INFINITY;
            }
            float y = sc[g][0][0];
#pragma unroll
            for (int e = 1; e < 8; e++) y = fmaxf(y, sc[g][e >> 2][e & 3]);
            mx[g] = CAP ? y : y * kf[g];
        }
    };
    // Probabilities of the scores of 32 keys from ts (step n), and their sums.  any:
    // some value is NaN, or all are far below the accumulators' reference (all zero,
    // say: their factor comes behind the sum, which would underflow with it).
    auto probs = [&](auto any_t, uint32_t ts, uint32_t n, Scores& sc, int32_t vref, bool vany) __attribute__((always_inline)) {
        constexpr bool ANY = decltype(any_t)::value;
        const bool far = ANY && oref - vref > 30;
        const float bias = kPBias + (far ? 0.0f : static_cast<float>(vref - oref));
        const float undelta = far ? 1.0f : pow2_field(127 + oref - vref);
#pragma unroll
        for (int g = 0; g < NCG; g++) {
            const float xf = CAP ? 1.0f : kf[g], off = bias - m[g];
            float p[8], sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                p[e] = fast_exp2(__builtin_fmaf(sc[g][e >> 2][e & 3], xf, off));
                sum += p[e];
            }
            l[g] = __builtin_fmaf(sum, undelta, l[g]);
            if (ANY && (far || vany)) {
                const float vscale = pow2_field(127 + vref - oref);
                const uint32_t nan = vany ? refs[n].nan[a4] : 0u;
                uint32_t t = ts + 4u * a4 - clo[g];
                asm volatile("" : "+v"(t));
#pragma unroll
                for (int e = 0; e < 8; e++) {  // a NaN value's readers' outputs are NaN
                    const bool bad = (nan >> e & 1u) & (t + (16u * (e >> 2) + (e & 3)) < cspan[g] ? 1u : 0u);
                    p[e] = bad ? NAN : far ? p[e] * vscale : p[e];
                }
            }
            if constexpr (PLO) {
                Ops<true>::split8_fast(p, ph[g], pl[g]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const f16x2 hh = __builtin_convertvector((f32x2{p[e], p[e + 1]}), f16x2);
                    ph[g][e] = hh[0];
                    ph[g][e + 1] = hh[1];
                }
            }
        }
    };

    if (S) {
        const bool on = wave < ng;  // (a wave without a group only moves)
        // References of the step whose scores are next (kn) and of the one whose
        // probabilities are (vr), requested a step early.
        uint32_t kn = refs[0].k, vr = refs[0].v;
        auto scale_of = [](uint32_t ref) { return __uint_as_float((ref - kQ8Up) << 23); };
        auto masked = [&](uint32_t ts) __attribute__((always_inline)) {  // some column does not read every key
            bool x = false;
#pragma unroll
            for (int g = 0; g < NCG; g++) x = x || ts < lomax[g] || ts + 32u > himin[g];
            return x;
        };
        auto one_step = [&](uint32_t n, Scores& sc, Scores& next) __attribute__((always_inline)) {
            const uint32_t ts = keys.first + 32u * n;
            const uint32_t v_now = vr;
            const float kscale = scale_of(kn);
            const int32_t vref = static_cast<int32_t>(v_now & 0x7fffffffu);
            vr = refs[min(n + 1u, S - 1u)].v;
            kn = refs[min(n + 2u, S - 1u)].k;
            bool rise = false;
#pragma unroll
            for (int g = 0; g < NCG; g++) rise = rise || mx[g] > m[g] + kTau;
            const bool risen = __builtin_amdgcn_ballot_w64(rise) != 0;
            const bool slow = risen || v_now >> 31 || vref > oref || oref - vref > 30 || masked(ts + 32u);
            // Behind the last step the scores of its keys follow again, unused.
            if (__builtin_expect(!slow, 1)) {
                qk(n + 1, next);
                order_reads<2 * KS, NCG*(QLO ? 2 : 1)>();
                probs(std::false_type{}, ts, n, sc, vref, false);
                pv(std::false_type{}, n);
                order_reads<MT, NCG*(PLO ? 2 : 1)>();
                maxima(std::false_type{}, ts + 32u, next, kscale);
                return;
            }
            float raise = 1.0f;
            if (vref > oref) {  // the accumulators' reference rises, two binades ahead
                raise = pow2_field(127 + oref - (vref + 2));
                oref = vref + 2;
            }
#pragma unroll
            for (int g = 0; g < NCG; g++) {
                const float top_g = col_max(mx[g]);
                const float to = top_g > m[g] + kTau ? top_g : m[g], f = fast_exp2(m[g] - to);
                l[g] *= f;
                alpha[g] = f * raise;
                m[g] = to;
            }
            qk(n + 1, next);
            order_reads<2 * KS, NCG*(QLO ? 2 : 1)>();
            probs(std::true_type{}, ts, n, sc, vref, v_now >> 31);
            pv(std::true_type{}, n);
            order_reads<MT, NCG*(PLO ? 2 : 1)>();
            if (masked(ts + 32u))
                maxima(std::true_type{}, ts + 32u, next, kscale);
            else
                maxima(std::false_type{}, ts + 32u, next, kscale);
        };
        // Step n reads K of step n + 1 and V of step n; what it requests, step n + 2,
        // goes where step n - 1 was, whose K was last read two barriers ago and whose
        // V one.
        wait_vm<0>();
        __syncthreads();
        if (on) {
            qk(0, sc0);
            maxima(std::true_type{}, keys.first, sc0, scale_of(kn));
            kn = refs[min(1u, S - 1u)].k;
        }
        for (uint32_t n = 0; n < S; n += 2) {
            request(n + 2);
            if (on) one_step(n, sc0, sc1);
            wait_vm<0>();
            __syncthreads();
            if (n + 1 == S) break;
            request(n + 3);
            if (on) one_step(n + 1, sc1, sc0);
            wait_vm<0>();
            __syncthreads();
        }
    }

    // Outputs: 4 consecutive dims a lane and unit (4 j + e: dims 64 j + 16 a4 + 4 e
    // ..), through LDS so that one loop over the units stores them.
    const float back = pow2_field(oref > 0 ? oref - static_cast<int32_t>(kQ8Up) : 127);  // (no step: nothing to undo)
    __syncthreads();
#pragma unroll
    for (int g = 0; g < NCG; g++) {
        l[g] = col_sum(l[g]);
        uint32_t row, head;
        const uint32_t item0 = column(g, con[g], row, head);
        const uint64_t pb = (static_cast<uint64_t>(item0 + part) * a.n_kvh + kvh) * kCols + c;
        const float inv = 1.0f / l[g];
#pragma unroll
        for (int j = 0; j < KB; j++) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                L.out[wave][e][lane] = __builtin_bit_cast(
                    u32x4, f32x4{o[g][4 * j][e], o[g][4 * j + 1][e], o[g][4 * j + 2][e], o[g][4 * j + 3][e]} * back);
#pragma unroll 1
            for (uint32_t e = 0; e < 4; e++) {
                const uint32_t d = 64u * j + 16u * a4 + 4u * e;
                if (!con[g] || d >= hd) continue;
                f32x4 v = __builtin_bit_cast(f32x4, L.out[wave][e][lane]);
                if (n_parts == 1) {
                    v = v * inv;
                    const float v4[4] = {v[0], v[1], v[2], v[3]};
                    store_y<4, true>(a, row, head, d, v4);
                } else {
                    publish_o(a.part_o + pb * HD + d, v);
                }
            }
        }
        if (!con[g]) continue;
        if (n_parts > 1 && a4 == 0) publish_ml(a.part_ml + 2 * pb, m[g], l[g]);
    }
}

bool args_query_lo(const AttnArgs& a) { return q8_query_lo(a.q_dt, a.rope_on); }

template <int HD, bool QLO, int PP>
void launch_q8_parts(dim3 grid, const AttnArgs& a, hipStream_t s) {
    constexpr int W = q8_waves(HD), NB = q8_ring(HD);
    if (a.full)
        hipLaunchKernelGGL((attn_q8<HD, W, NB, QLO, PP, true>), grid, dim3(64 * W), 0, s, a);
    else
        hipLaunchKernelGGL((attn_q8<HD, W, NB, QLO, PP, false>), grid, dim3(64 * W), 0, s, a);
}

template <int HD>
void launch_q8_hd(dim3 grid, const AttnArgs& a, hipStream_t s) {
    const bool lo = args_query_lo(a), f32 = a.y_dt == THB_DT_F32;
    if (lo)
        f32 ? launch_q8_parts<HD, true, 3>(grid, a, s) : launch_q8_parts<HD, true, 2>(grid, a, s);
    else
        f32 ? launch_q8_parts<HD, false, 3>(grid, a, s) : launch_q8_parts<HD, false, 2>(grid, a, s);
}

template <int HD, int NCG, bool QLO, bool PLO>
void launch_q8_prefill_cap(dim3 grid, const AttnArgs& a, hipStream_t s) {
    if (a.cap2 != 0.0f)
        hipLaunchKernelGGL((attn_q8_prefill<HD, NCG, QLO, PLO, true>), grid, dim3(64 * kQ8PrefillWaves), 0, s, a);
    else
        hipLaunchKernelGGL((attn_q8_prefill<HD, NCG, QLO, PLO, false>), grid, dim3(64 * kQ8PrefillWaves), 0, s, a);
}

template <int HD, int NCG, bool QLO>
void launch_q8_prefill_out(dim3 grid, const AttnArgs& a, hipStream_t s) {
    a.y_dt == THB_DT_F32 ? launch_q8_prefill_cap<HD, NCG, QLO, true>(grid, a, s)
                         : launch_q8_prefill_cap<HD, NCG, QLO, false>(grid, a, s);
}

}  // namespace

void launch_q8_expand(uint32_t hd, const AttnArgs& a, hipStream_t s) {
    const dim3 grid(a.steps, a.n_kvh);
    if (hd == 64)
        hipLaunchKernelGGL(q8_expand<64>, grid, dim3(128), 0, s, a);
    else
        hipLaunchKernelGGL(q8_expand<128>, grid, dim3(256), 0, s, a);
}

void launch_q8_prefill(uint32_t hd, uint32_t ncg, dim3 grid, const AttnArgs& a, hipStream_t s) {
    const bool lo = args_query_lo(a);
    if (hd == 64)
        lo ? launch_q8_prefill_out<64, 1, true>(grid, a, s) : launch_q8_prefill_out<64, 1, false>(grid, a, s);
    else if (lo)
        launch_q8_prefill_out<128, 1, true>(grid, a, s);
    else
        ncg == 2 ? launch_q8_prefill_out<128, 2, false>(grid, a, s) : launch_q8_prefill_out<128, 1, false>(grid, a, s);
}

void launch_q8_decode(uint32_t hd, dim3 grid, const AttnArgs& a, hipStream_t s) {
    switch (hd) {
        case 64: launch_q8_hd<64>(grid, a, s); break;
        case 128: launch_q8_hd<128>(grid, a, s); break;
        case 256: launch_q8_hd<256>(grid, a, s); break;
        default: launch_q8_hd<512>(grid, a, s); break;
    }
}

}  // namespace thb
