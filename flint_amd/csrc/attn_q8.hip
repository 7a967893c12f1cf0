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

// ---------------------------------------------------------------- chunks
// Prefill blocks.  One workgroup of 8 waves handles a block of query groups for
// one KV head and one partition of the block's keys; wave w takes groups w, w +
// 8, ..., up to NCG of them (16 query vectors each).  Keys go in tiles of 64:
// the codes of the next tile are requested from memory before this one's
// products, converted to f16 behind them and written to the other of two LDS
// buffers in operand order (16 bytes a lane, no bank conflicts), so a code is
// converted once per workgroup and every operand read feeds NCG products.
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
// 16-bit output (2^-12 of each, below the output's own rounding) or split into
// two for f32 (PLO).  The sum l is taken from the unrounded ones.
constexpr float kPBias = 7.0f;
constexpr uint32_t kQ8Tile = 64, kQ8Up = 7;

template <int HD>
struct Q8PrefillLds {
    u32x4 k[2][kQ8Tile / 16][HD / 32][64];  // [16-key tile][k-step]
    u32x4 v[2][kQ8Tile / 32][HD / 16][64];  // [32-key step][output tile]
    uint32_t page[kMaxPartPages];
    uint32_t kref[2][kQ8Tile / 32], vref[2][kQ8Tile / 32];
    uint32_t vnan[2][kQ8Tile / 32][4];  // NaN values among a lane group's 8 keys of a step, a bit each
    uint32_t vany[2][kQ8Tile / 32];
};

// 2^n for an exponent field, 0 below the normal range.
__device__ __forceinline__ float pow2_field(int32_t field) {
    return __uint_as_float(field > 0 ? static_cast<uint32_t>(field) << 23 : 0u);
}
// Maximum over the 16 lanes of a lane group / over the 4 lane groups.
__device__ __forceinline__ uint32_t max16(uint32_t x) {
#pragma unroll
    for (int i = 1; i < 16; i <<= 1) x = max(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), i)));
    return x;
}
__device__ __forceinline__ uint32_t max_groups(uint32_t x) {
    x = max(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), 16)));
    return max(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), 32)));
}

template <int HD, int NCG, bool QLO, bool PLO, bool CAP>
__global__ __launch_bounds__(512, 2) void attn_q8_prefill(AttnArgs a) {
    constexpr int W = 8;
    constexpr int KS = HD / 32, KB = HD / 64, MT = HD / 16;
    constexpr int NS = kQ8Tile / 32;             // 32-key steps a tile
    constexpr int TASKS = 2 * NS * KB;           // staging: (operand, step, block) a wave
    constexpr int TPW = (TASKS + W - 1) / W;
    __shared__ Q8PrefillLds<HD> L;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t a4 = lane >> 4, c = lane & 15u;
    const uint32_t item = blockIdx.x / a.n_kvh, kvh = blockIdx.x - item * a.n_kvh;
    const uint32_t* B = a.bitems + static_cast<uint64_t>(item) * kBItemWords;
    const uint32_t g0 = B[0], ng = B[1], seq = B[2], part = B[kBlockWords];
    const uint32_t n_parts = B[5], P = B[7], pbeg = B[6] + part * P;
    const BlockKeys keys = block_keys(B[3], B[4], pbeg, P, kQ8Tile);
    const uint32_t tb = keys.tb, te = keys.te;
    const uint32_t hd = a.head_dim, width = q8_width(hd), nb = width >> 6;
    const uint32_t pshift = a.page_shift, pmask = (1u << pshift) - 1u;
    const uint32_t lp0 = pbeg >> pshift;
    {
        const uint32_t npg = P >> pshift;
        const uint32_t* trow = a.table + static_cast<uint64_t>(seq) * a.max_pages;
        for (uint32_t i = tid; i < npg; i += 64 * W) {
            const uint32_t lp = lp0 + i;
            const bool used = tb < te && (lp << pshift) < te && ((lp + 1) << pshift) > tb;
            const uint32_t pg = used ? trow[lp] : 0u;
            L.page[i] = pg < a.pages ? pg : 0u;
        }
    }

    // This wave's groups and columns; [wlo, whi) spans their keys.
    bool con[NCG];
    uint32_t row[NCG], head[NCG], clo[NCG], cspan[NCG], item0[NCG], lomax[NCG], himin[NCG];
    uint32_t wlo = 0xFFFFFFFFu, whi = 0;
    f16x8 qh[NCG][KS], ql[NCG][QLO ? KS : 1];
    float qf[NCG];
#pragma unroll
    for (int g = 0; g < NCG; g++) {
        const uint32_t gi = wave + W * g;
        const bool gon = gi < ng;
        const uint32_t* G = a.groups + (g0 + (gon ? gi : 0u)) * kGroupWords;
        const uint32_t r0 = G[0], R = G[1], h0 = G[2], H = G[3];
        item0[g] = G[10];
        con[g] = gon && c < R * H;
        const uint32_t rr = con[g] ? c / H : 0u;
        row[g] = r0 + rr;
        head[g] = kvh * a.nq_per_kv + h0 + (con[g] ? c - rr * H : 0u);
        const uint32_t lo = con[g] ? max(a.ranges[2 * row[g]], tb) : 0u;
        const uint32_t hi = con[g] ? min(a.ranges[2 * row[g] + 1], te) : 0u;
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
        const uint32_t glo = max(G[5], tb), ghi = min(G[6], te);
        if (gon && glo < ghi) {
            wlo = min(wlo, glo);
            whi = max(whi, ghi);
        }
        // The sign of the score scale goes into the query, its size into qf >= 0.
        const float undo = load_q_scaled<KS, QLO, true>(a, con[g], row[g], head[g], a4, qh[g], ql[g], a.qpre);
        qf[g] = undo * a.qpost;
    }

    // Staging of one tile: task = operand, step s, block j; a lane's 16 bytes of
    // the step's two 16-key tiles, their scales.
    const uint8_t* kcodes = reinterpret_cast<const uint8_t*>(a.k);
    const uint8_t* vcodes = reinterpret_cast<const uint8_t*>(a.v);
    const uint32_t first16 = tb & ~15u, last16 = te > tb ? (te - 1u) & ~15u : 0u;
    struct Stage {
        u32x4 codes[2];
        uint32_t scale[2];
    };
    auto fetch = [&](uint32_t t0, Stage (&x)[TPW]) {
#pragma unroll
        for (uint32_t i = 0; i < TPW; i++) {
            const uint32_t task = wave + W * i;
            if (task >= TASKS) break;
            const bool is_v = task >= TASKS / 2;
            const uint32_t r = task - (is_v ? TASKS / 2 : 0u), s = r / KB, j = r - s * KB;
#pragma unroll
            for (uint32_t h = 0; h < 2; h++) {
                const uint32_t t = min(max(t0 + 32u * s + 16u * h, first16), last16);
                const uint32_t page = __builtin_amdgcn_readfirstlane(L.page[(t >> pshift) - lp0]);
                const uint64_t slot = ((static_cast<uint64_t>(kvh) * a.pages + page) << pshift) + (t & pmask);
                const uint32_t at = (j < nb ? j << 10 : 0u) + 16u * lane;
                const uint8_t* sc = a.scales + slot * 2u;
                x[i].codes[h] = *reinterpret_cast<const u32x4*>((is_v ? vcodes : kcodes) + slot * width + at);
                if (is_v)
                    x[i].scale[h] = *reinterpret_cast<const uint32_t*>(sc + 8u * a4 + 4u);
                else
                    x[i].scale[h] = sc[(c >> 2) * 8u + (c & 3u)];
            }
        }
    };
    auto stage = [&](uint32_t buf, const Stage (&x)[TPW]) {
#pragma unroll
        for (uint32_t i = 0; i < TPW; i++) {
            const uint32_t task = wave + W * i;
            if (task >= TASKS) break;
            const bool is_v = task >= TASKS / 2;
            const uint32_t r = task - (is_v ? TASKS / 2 : 0u), s = r / KB, j = r - s * KB;
            if (!is_v) {
                const uint32_t b0 = x[i].scale[0], b1 = x[i].scale[1];
                const uint32_t ref = max(max16(max(b0 == 255u ? 0u : b0, b1 == 255u ? 0u : b1)), kQ8Up + 1u);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t b = h ? b1 : b0;
                    const float f = pow2_field(127 + static_cast<int32_t>(kQ8Up) + static_cast<int32_t>(b) -
                                               static_cast<int32_t>(ref));
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        u32x4 w;
#pragma unroll
                        for (int d = 0; d < 2; d++) {
                            const uint32_t cw = x[i].codes[h][2 * q + d];
                            w[2 * d] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(cw, f, false));
                            w[2 * d + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(cw, f, true));
                        }
                        if (b == 255u) w = u32x4{0x7E007E00u, 0x7E007E00u, 0x7E007E00u, 0x7E007E00u};  // a NaN key
                        L.k[buf][2 * s + h][2 * j + q][lane] = w;
                    }
                }
                if (j == 0 && lane == 0) L.kref[buf][s] = ref;
            } else {
                uint32_t ref = 0u, nan = 0u;
                uint32_t bb[2][4];
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t b = (x[i].scale[h] >> (8 * e)) & 255u;
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
                        f[h][e >> 1][e & 1] = static_cast<_Float16>(
                            pow2_field(127 + static_cast<int32_t>(kQ8Up) + static_cast<int32_t>(bb[h][e]) -
                                       static_cast<int32_t>(ref)));
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    u32x4 w;
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            const f16x2 v2 = q ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[i].codes[h][d], 1.0f, true)
                                               : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[i].codes[h][d], 1.0f, false);
                            w[2 * h + q] = __builtin_bit_cast(uint32_t, v2 * f[h][q]);
                        }
                    L.v[buf][s][4 * j + d][lane] = w;
                }
                if (j == 0) {
                    const bool any = __builtin_amdgcn_ballot_w64(nan != 0u) != 0;
                    if (c == 0) L.vnan[buf][s][a4] = nan;
                    if (lane == 0) {
                        L.vref[buf][s] = ref;
                        L.vany[buf][s] = any;
                    }
                }
            }
        }
    };

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

    auto step = [&](uint32_t buf, uint32_t s, uint32_t ts) {
        const int32_t kref = __builtin_amdgcn_readfirstlane(L.kref[buf][s]);
        const int32_t vref = __builtin_amdgcn_readfirstlane(L.vref[buf][s]);
        const bool vany = __builtin_amdgcn_readfirstlane(L.vany[buf][s]) != 0u;
        f32x4 sc[NCG][2];
#pragma unroll
        for (int g = 0; g < NCG; g++) sc[g][0] = sc[g][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < KS; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const f16x8 kc = __builtin_bit_cast(f16x8, L.k[buf][2 * s + h][j][lane]);
#pragma unroll
                for (int g = 0; g < NCG; g++) {
                    sc[g][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, qh[g][j], sc[g][h], 0, 0, 0);
                    if constexpr (QLO) sc[g][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, ql[g][j], sc[g][h], 0, 0, 0);
                }
            }
        if (vref > oref) {  // the accumulators' reference rises, two binades ahead
            const float f = pow2_field(127 + oref - (vref + 2));
#pragma unroll
            for (int g = 0; g < NCG; g++)
#pragma unroll
                for (int i = 0; i < MT; i++) o[g][i] *= f;
            oref = vref + 2;
        }
        // Values far below the reference (all zero, say): their factor is applied
        // behind the sum, which would underflow with it.
        const bool far = oref - vref > 30;
        const float delta = static_cast<float>(vref - oref), vscale = pow2_field(127 + vref - oref);
        const float undelta = far ? 1.0f : pow2_field(127 + oref - vref);
        const float kscale = __uint_as_float(static_cast<uint32_t>(kref - static_cast<int32_t>(kQ8Up)) << 23);
        f16x8 ph[NCG], pl[PLO ? NCG : 1];
#pragma unroll
        for (int g = 0; g < NCG; g++) {
            const float kf = qf[g] * kscale;
            const bool mask = ts < lomax[g] || ts + 32u > himin[g];
            float x[8], mx;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[e] = sc[g][e >> 2][e & 3];
                if constexpr (CAP) x[e] = cap2 * tanh_approx(x[e] * kf);
            }
            if (mask) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t t = ts + 16u * (e >> 2) + 4u * a4 + (e & 3);
                    x[e] = t - clo[g] < cspan[g] ? x[e] : -INFINITY;
                }
            }
            mx = x[0];
#pragma unroll
            for (int e = 1; e < 8; e++) mx = fmaxf(mx, x[e]);
            const float xf = CAP ? 1.0f : kf;
            // (-inf * 0 where a column has no key or no scale: no maximum.)
            mx = mx == -INFINITY ? mx : mx * xf;
            if (__builtin_amdgcn_ballot_w64(mx > m[g] + kTau) != 0) {
                mx = col_max(mx);
                if (mx > m[g] + kTau) {
                    const float alpha = fast_exp2(m[g] - mx);
                    l[g] *= alpha;
#pragma unroll
                    for (int i = 0; i < MT; i++) o[g][i] *= alpha;
                    m[g] = mx;
                }
            }
            const float off = kPBias + (far ? 0.0f : delta) - m[g];
            float p[8], sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                // (a masked score stays -inf whatever the factor)
                const float y = mask && x[e] == -INFINITY ? -INFINITY : __builtin_fmaf(x[e], xf, off);
                p[e] = fast_exp2(y);
                sum += p[e];
            }
            l[g] = __builtin_fmaf(sum, undelta, l[g]);
            if (far) {
#pragma unroll
                for (int e = 0; e < 8; e++) p[e] *= vscale;
            }
            if (vany) {  // a NaN value among the step's: its readers' outputs are NaN
                const uint32_t nan = L.vnan[buf][s][a4];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint32_t t = ts + 16u * (e >> 2) + 4u * a4 + (e & 3);
                    if ((nan >> e & 1u) && t - clo[g] < cspan[g]) p[e] = NAN;
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
#pragma unroll
        for (int i = 0; i < MT; i++) {
            const f16x8 vc = __builtin_bit_cast(f16x8, L.v[buf][s][i][lane]);
#pragma unroll
            for (int g = 0; g < NCG; g++) {
                o[g][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, ph[g], o[g][i], 0, 0, 0);
                if constexpr (PLO) o[g][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vc, pl[g], o[g][i], 0, 0, 0);
            }
        }
    };

    __syncthreads();  // the page list
    if (keys.tiles) {
        Stage x[TPW];
        fetch(keys.first, x);
        stage(0, x);
        __syncthreads();
        for (uint32_t i = 0; i < keys.tiles; i++) {
            const uint32_t t0 = keys.first + kQ8Tile * i;
            const bool more = i + 1 < keys.tiles;
            if (more) fetch(t0 + kQ8Tile, x);
#pragma unroll
            for (uint32_t s = 0; s < NS; s++) {
                const uint32_t ts = t0 + 32u * s;
                if (ts < whi && ts + 32u > wlo) step(i & 1u, s, ts);
            }
            if (more) stage((i + 1u) & 1u, x);
            __syncthreads();
        }
    }

    const float back = pow2_field(oref > 0 ? oref - static_cast<int32_t>(kQ8Up) : 127);  // (no step: nothing to undo)
#pragma unroll
    for (int g = 0; g < NCG; g++) {
        l[g] = col_sum(l[g]);
        if (!con[g]) continue;
        const uint64_t pb = (static_cast<uint64_t>(item0[g] + part) * a.n_kvh + kvh) * kCols + c;
#pragma unroll
        for (int j = 0; j < KB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t d = 64u * j + 16u * a4 + 4u * e;
                if (d >= hd) continue;
                f32x4 v = f32x4{o[g][4 * j][e], o[g][4 * j + 1][e], o[g][4 * j + 2][e], o[g][4 * j + 3][e]} * back;
                if (n_parts == 1) {
                    v = v * (1.0f / l[g]);
                    const float v4[4] = {v[0], v[1], v[2], v[3]};
                    store_y<4, true>(a, row[g], head[g], d, v4);
                } else {
                    publish_o(a.part_o + pb * HD + d, v);
                }
            }
        if (n_parts > 1 && a4 == 0) publish_ml(a.part_ml + 2 * pb, m[g], l[g]);
    }
}

bool args_query_lo(const AttnArgs& a) { return q8_query_lo(a.q_dt, a.rope_on); }

template <int HD>
void launch_q8_hd(dim3 grid, const AttnArgs& a, hipStream_t s) {
    constexpr int W = q8_waves(HD), NB = q8_ring(HD);
    const bool lo = args_query_lo(a);
    if (a.full && lo)
        hipLaunchKernelGGL((attn_q8<HD, W, NB, true, true>), grid, dim3(64 * W), 0, s, a);
    else if (a.full)
        hipLaunchKernelGGL((attn_q8<HD, W, NB, false, true>), grid, dim3(64 * W), 0, s, a);
    else if (lo)
        hipLaunchKernelGGL((attn_q8<HD, W, NB, true, false>), grid, dim3(64 * W), 0, s, a);
    else
        hipLaunchKernelGGL((attn_q8<HD, W, NB, false, false>), grid, dim3(64 * W), 0, s, a);
}

template <int HD, int NCG, bool QLO, bool PLO>
void launch_q8_prefill_cap(dim3 grid, const AttnArgs& a, hipStream_t s) {
    if (a.cap2 != 0.0f)
        hipLaunchKernelGGL((attn_q8_prefill<HD, NCG, QLO, PLO, true>), grid, dim3(512), 0, s, a);
    else
        hipLaunchKernelGGL((attn_q8_prefill<HD, NCG, QLO, PLO, false>), grid, dim3(512), 0, s, a);
}

template <int HD, bool QLO, bool PLO>
void launch_q8_prefill_ncg(uint32_t ncg, dim3 grid, const AttnArgs& a, hipStream_t s) {
    constexpr int NCG = static_cast<int>(q8_groups(HD, QLO));
    if (ncg == 1) return launch_q8_prefill_cap<HD, 1, QLO, PLO>(grid, a, s);
    if constexpr (NCG >= 2) {
        if (ncg == 2) return launch_q8_prefill_cap<HD, 2, QLO, PLO>(grid, a, s);
    }
    if constexpr (NCG >= 3) return launch_q8_prefill_cap<HD, 3, QLO, PLO>(grid, a, s);
}

template <int HD>
void launch_q8_prefill_hd(uint32_t ncg, dim3 grid, const AttnArgs& a, hipStream_t s) {
    const bool plo = a.y_dt == THB_DT_F32;
    if (args_query_lo(a))
        plo ? launch_q8_prefill_ncg<HD, true, true>(ncg, grid, a, s)
            : launch_q8_prefill_ncg<HD, true, false>(ncg, grid, a, s);
    else
        plo ? launch_q8_prefill_ncg<HD, false, true>(ncg, grid, a, s)
            : launch_q8_prefill_ncg<HD, false, false>(ncg, grid, a, s);
}

}  // namespace

void launch_q8_prefill(uint32_t hd, uint32_t ncg, dim3 grid, const AttnArgs& a, hipStream_t s) {
    switch (hd) {
        case 64: launch_q8_prefill_hd<64>(ncg, grid, a, s); break;
        case 128: launch_q8_prefill_hd<128>(ncg, grid, a, s); break;
        default: launch_q8_prefill_hd<256>(ncg, grid, a, s); break;
    }
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
