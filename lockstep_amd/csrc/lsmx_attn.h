// Arguments and device helpers shared by the attention kernels
// (attention.hip, attention_bwd.hip, kv_cache.hip).
//
// Visibility, everywhere: the query of token position p sees key j when
// 0 <= j <= p and (no window, or j > p - window, or j < sinks).
#pragma once

#include "lsmx_common.h"
#include "lsmx_internal.h"

namespace lsmx {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct Vec;
template <>
struct Vec<__bf16> {
    typedef bf16x4 x4;
    typedef bf16x8 x8;
};
template <>
struct Vec<_Float16> {
    typedef f16x4 x4;
    typedef f16x8 x8;
};

// C (16 x 16, fp32) += A (16 x 32) B (32 x 16).  Lane 16g + r holds A[r][8g..8g+7],
// B[8g..8g+7][r] and C[4g..4g+3][r].
LSMX_DEV f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
LSMX_DEV f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Position of 16-byte chunk c of row r in an LDS tile of NC chunks per row
// (8 or 16).  The 16 rows that one operand read touches are put on 16 different
// 16-byte bank groups, and so are the 8 rows x 2 chunks of half a transposing
// read.  The counters still show a conflict cycle for every three LDS cycles
// (forward 8.2 of 24.5 million, dQ 16.6 of 34, dK and dV 22.7 of 60): not all reads
// are served in the groups assumed here.
template <int NC>
LSMX_DEV int swz(int r, int c) {
    if constexpr (NC == 16) return c ^ (((r & 7) << 1) | ((r >> 3) & 1));
    const int j = (r >> 1) & 7;
    return c ^ (((j & 3) << 1) | (j >> 2));
}

// The transposing LDS read: lane 16g + r gets element r of a 16-element run
// of rows 4g' .. 4g'+3, given the address of row 4g' + r / 4, element 4 (r % 4).
template <typename T>
LSMX_DEV typename Vec<T>::x4 read_tr(const T *p) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    return __builtin_bit_cast(typename Vec<T>::x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p));
}

template <typename X4, typename X8>
LSMX_DEV X8 join(X4 a, X4 b) {
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The mask, without branches; low is the last key that the window hides
// (window_low).
LSMX_DEV bool sees(int j, int pos, int low, int sinks) { return (j <= pos) & ((j > low) | (j < sinks)); }
LSMX_DEV int window_low(int pos, int window) { return window ? pos - window : -1; }

// max and sum over the 4 lanes 16 apart that share a row, by register swaps
// between 16-lane rows (two VALU operations; a shuffle goes through LDS).
LSMX_DEV float max_rows(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
    x = fmaxf(u2f(a[0]), u2f(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
    return fmaxf(u2f(b[0]), u2f(b[1]));
}
LSMX_DEV float sum_rows(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
    x = u2f(a[0]) + u2f(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
    return u2f(b[0]) + u2f(b[1]);
}
LSMX_DEV int lane_of(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
LSMX_DEV int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// n / d for n < 2^31 by multiplication: m = ceil(2^(31 + L) / d), L = ceil(log2 d),
// sh = L - 1 (d = 1: n itself).
struct FastDiv {
    uint32_t d, m, sh;
};
inline FastDiv fast_div(uint32_t d) {
    uint32_t L = 0;
    while ((1u << L) < d) ++L;
    return {d, (uint32_t)((((uint64_t)1 << (31 + L)) + d - 1) / d), L ? L - 1 : 0};
}
LSMX_DEV int div_by(int n, FastDiv f) { return f.d == 1 ? n : (int)(__umulhi((uint32_t)n, f.m) >> f.sh); }

struct AttnArgs {
    const void *q, *k, *v;
    void *o;
    float *lse;  // base 2: m c + log2(sum), c = scale log2(e)
    int batch, heads, kv_heads, group, dim;
    int q_len, k_len;                                    // dense
    int64_t q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h;  // strides, in elements
    int64_t o_b, o_t, o_h, lse_b, lse_h;
    const int32_t *offsets;  // packed sequences: [batch + 1], else null
    int tokens;              // packed: tokens in all
    int window, sinks;       // window 0: none (then sinks is 0)
    float c;                 // scale * log2(e)
    FastDiv by_group;
    int tiles, run;  // tiles per kv head over all sequences (dense: of one sequence times batch); items per XCD, or 0: see item_of
    // backward
    const void *d_o;
    int64_t do_b, do_t, do_h;
    float *delta;
    void *dq, *dk, *dv;  // contiguous, laid out as q, k, v
    float scale;
    void *o_lo;          // o as computed less o as rounded, laid out as o (forward: null to leave out)
    float *part;         // far rows' partial gradients of the sinks
    int chunk, far_slots;  // rows of a chunk (0: no far rows apart), chunks of all sequences
    float *share_part;     // dK and dV of each share of a key tile's rows: [share][dK, dV][key][kv head][dim]
    int shares, share_rows;  // shares > 1: most of a tile, rows of one
};

// The item of a workgroup: a tile of one key head, and one of `shares` shares.
// Ids go to the 8 XCDs in turn.  A multiple of 8 key heads: `run` items in order on
// each, so that its L2 holds one head's keys after the other.  Else the heads are
// the ids' fastest part: an XCD still has one or few of them (4: one), all
// XCDs long tiles and short ones, and the short come last (in runs an XCD had
// the half of a head with the long rows: 5086 tokens of 32/4 heads of 128, causal,
// 419 us against 303; 5506 of 5/1 heads of 64, 82 against 64).  The grid
// is padded; items past the last are dropped by the caller.
struct Item {
    int tile, head, share;
};
LSMX_DEV Item item_of(const AttnArgs &a, int shares) {
    const int id = blockIdx.x;
    if (a.run) {
        const int item = (id & 7) * a.run + (id >> 3), rest = item / a.tiles, head = rest / shares;
        return Item{item - rest * a.tiles, head, rest - head * shares};
    }
    const int rest = id / a.kv_heads, share = rest / a.tiles;
    return Item{rest - share * a.tiles, share < shares ? id - rest * a.kv_heads : a.kv_heads, share};
}
inline unsigned order_items(AttnArgs &a, int64_t items) {
    a.run = a.kv_heads % 8 ? 0 : (int)((items + 7) / 8);
    return (unsigned)(a.run ? a.run * 8 : items);
}

// One sequence of a packed or dense batch.
struct Seq {
    int b, q_len, k_len, shift;  // query token t has position t + shift
    int64_t q0, k0;              // first token (packed: in the token axis, else 0)
    int tile;
    int idx;                     // packed: its place in the order of tiles
};

// The sequence and tile of work tile t, tiles of `size` rows with `mult` rows
// per token, `len` tokens in a dense sequence.  Packed tokens before offsets[0] and from offsets[batch] on
// belong to two more sequences that see nothing (k_len 0).
// Returns false past the last tile.
LSMX_DEV bool find_tile(const AttnArgs &a, int t, int size, int mult, int len, Seq &s) {
    t = uniform(t);
    if (!a.offsets) {
        const int per = (len * mult + size - 1) / size;
        s.b = t / per;
        if (s.b >= a.batch) return false;
        s.tile = t - s.b * per;
        s.q_len = a.q_len;
        s.k_len = a.k_len;
        s.shift = a.k_len - a.q_len;
        s.q0 = s.k0 = 0;
        return true;
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int first = 0; first < a.batch + 2; first += 64) {
        const int i = first + lane;
        int lo = 0, hi = 0;
        if (i < a.batch + 2) {
            lo = i == 0 ? 0 : min(max(a.offsets[i - 1], 0), a.tokens);
            hi = i == a.batch + 1 ? a.tokens : min(max(a.offsets[i], 0), a.tokens);
        }
        const int own = max(hi - lo, 0);
        const int n = (int)(((int64_t)own * mult + size - 1) / size);
        int upto = n;
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(upto, d);
            if (lane >= d) upto += x;
        }
        const uint64_t hit = __ballot(before + upto > t);
        if (hit) {
            const int w = __ffsll((unsigned long long)hit) - 1;
            s.tile = t - before - (lane_of(upto, w) - lane_of(n, w));
            s.q_len = lane_of(own, w);
            s.q0 = s.k0 = lane_of(lo, w);
            const int idx = s.idx = first + w;
            s.b = 0;
            s.k_len = idx >= 1 && idx <= a.batch ? s.q_len : 0;
            s.shift = s.k_len ? 0 : -s.q_len;  // dead sequence: positions below 0
            return true;
        }
        before += lane_of(upto, 63);
    }
    return false;
}

// A paged MXFP4 cache: pool of pages [pages][kv_heads][page][..], codes D / 2
// and E8M0 scales D / 32 bytes per vector; block tables and lengths of the
// sequences.  A page id outside the pool and a position past the table are
// never followed: their keys are hidden.
struct Pool {
    uint8_t *kc, *ks, *vc, *vs;
    const int32_t *table, *lengths;
    int pages, kv_heads, dim, page, page_shift, max_pages;

    LSMX_DEV int length(int b) const {
        return __builtin_amdgcn_readfirstlane(min(max(lengths[b], 0), max_pages << page_shift));
    }
    // the page of position j of sequence b, or -1
    LSMX_DEV int page_of(int b, int j) const {
        const int p = table[(int64_t)b * max_pages + (j >> page_shift)];
        return (uint32_t)p < (uint32_t)pages ? p : -1;
    }
    // vector index (in units of one token's head vector) of position j in page p
    LSMX_DEV int64_t vec(int p, int h, int j) const {
        return (((int64_t)p * kv_heads + h) << page_shift) + (j & (page - 1));
    }
};

// Attention of the newest q_len tokens of every sequence over the cache.
struct AttendArgs {
    AttnArgs a;  // q, o, lse, strides, mask and scale; k_len and the rest unused
    Pool p;
    float *weights;       // [batch, kv_heads, w_len], or null
    int64_t w_len;
    int splits;           // shares of the keys, each with workgroups of its own
    float *part, *part_m; // their sums: [batch kv_heads splits rows][DP] and [..][2]
};

struct AppendArgs {
    const void *k, *v;
    int64_t k_t, k_h, v_t, v_h;  // strides, in elements
    Pool p;
    int batch, tokens, per_seq;  // per_seq: tokens of each sequence, packed with offsets: 0
    const int32_t *offsets;
    FastDiv by_seq;
    void *k_out, *v_out;         // bf16 values [tokens, kv_heads, dim], or null
};

struct EvictArgs {
    Pool p;
    const int32_t *out_table;
    int out_max_pages;
    const float *weights;
    int64_t w_len;
    int batch, keep, sinks, recent;
    int32_t *index, *new_lengths;
    float *new_weights;
};

// Probabilities enter the product with the values relative to their row's
// largest so far.  fp16 holds 2^-24 to 65504, so there they are lifted by
// 2^kLift, with the sum of their row: one of 2^-25 still has all its bits, and what
// a lost one leaves out is at most 2^-36 of the largest.  bf16 has fp32's range.
template <typename T>
constexpr float kLift = __is_same(T, _Float16) ? 11.f : 0.f;

// The 8 elements of four bytes of codes, times their block's scale.  Exact in bf16,
// which has E8M0's range; in fp16 where it holds them (holds).
LSMX_DEV bf16x8 fp4x8_to(uint32_t w, float sc, bf16x8) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
LSMX_DEV f16x8 fp4x8_to(uint32_t w, float sc, f16x8) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 1);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 3);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
template <typename T>
LSMX_DEV typename Vec<T>::x8 fp4x8(uint32_t w, float sc) {
    return fp4x8_to(w, sc, typename Vec<T>::x8{});
}

// Rows in fp16 take the cached values in fp16 too (as bf16 operands they would need
// two terms of everything, and 1.5 times as long), where it has all elements of a
// block: 6 times 2^13 is the largest it holds, half of 2^-23 the smallest.  A cache
// written from fp16 has no other blocks but those whose largest value is below 2^-21; one
// written from bf16 may have any.  A workgroup that meets one takes its rows in
// fp32 without matrix instructions (attend_exact), 20 to 80 times as long: 64 x 8192
// tokens of 8 key heads of 128, 4 rows, 2.3 ms for 90 us.  A second form of the
// kernels' loops with bf16 operands would be faster there, and cost the others a wave
// per SIMD.
template <typename T>
LSMX_DEV bool holds(uint32_t e8m0) {
    return !__is_same(T, _Float16) || e8m0 - (127u - 23u) <= 36u;
}

// The scale of a block that T holds (of others anything: their products are not used).
template <typename T>
LSMX_DEV float block_scale(uint32_t e8m0) {
    if constexpr (__is_same(T, _Float16)) return u2f(e8m0 << 23);
    return e8m0_to_f32(e8m0);
}

// The product of a row with a cached vector, in fp32.
template <typename T>
LSMX_DEV float dot_exact(const T *q, const uint8_t *codes, const uint8_t *scale, int dim) {
    float sum = 0.f;
#pragma unroll 1
    for (int d = 0; d < dim; d += 8) {
        const typename Vec<T>::x8 x = *(const typename Vec<T>::x8 *)(q + d);
        const bf16x8 k = fp4x8<__bf16>(*(const uint32_t *)(codes + d / 2), e8m0_to_f32(scale[d >> 5]));
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = __builtin_fmaf((float)x[i], (float)k[i], sum);
    }
    return sum;
}

// Attention of rows [row0, row1) of sequence b and key head hkv over the keys of
// `tiles` tiles of TS keys, the i-th from key key_of(i) on; writes what the kernels
// write of a share.  A wave takes a row: its lanes the keys for the scores, then the
// head's elements for the values.
template <typename T, int DP, int TS, typename F>
LSMX_DEV void attend_exact(const AttendArgs &x, int b, int hkv, int share, int row0, int row1, int tiles, F key_of) {
    constexpr int NE = DP / 64;
    const AttnArgs &a = x.a;
    const Pool &p = x.p;
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));  // nothing made from it is shared with the caller's loop, and held over that
    const int lane = thread & 63, len = p.length(b), rows = a.q_len * a.group;
#pragma unroll 1
    for (int row = row0 + uniform(thread >> 6); row < row1; row += blockDim.x >> 6) {
        const int tok = div_by(row, a.by_group), h = hkv * a.group + row - tok * a.group, pos = tok + len - a.q_len;
        const int low = window_low(pos, a.window);
        const T *q = (const T *)a.q + b * a.q_b + tok * a.q_t + h * a.q_h;
        float m = -INFINITY, l = 0.f, acc[NE] = {};
#pragma unroll 1
        for (int i = 0; i < tiles; ++i) {
            const int j = key_of(i) + lane;
            int pg = -1;
            if (lane < TS && j < len && sees(j, pos, low, a.sinks)) pg = p.page_of(b, j);
            const int64_t vec = p.vec(max(pg, 0), hkv, max(j, 0));
            const float s = pg >= 0 ? dot_exact(q, p.kc + vec * (DP / 2), p.ks + vec * (DP / 32), DP) : -INFINITY;
            float top = s;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
            top = fmaxf(top, m);
            const float alpha = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - top) * a.c);
            const float w = pg < 0 ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(s, a.c, top == -INFINITY ? 0.f : kLift<T> - top * a.c));
            m = top;
            l = __builtin_fmaf(l, alpha, w);
#pragma unroll
            for (int e = 0; e < NE; ++e) acc[e] *= alpha;
#pragma unroll 1
            for (int t = 0; t < TS; ++t) {
                const int pt = lane_of(pg, t);
                if (pt < 0) continue;
                const float wt = u2f(lane_of(f2u(w), t));
                const int64_t v = p.vec(pt, hkv, lane_of(j, t));
                const uint32_t code = p.vc[v * (DP / 2) + lane * NE / 2] >> (NE == 1 ? 4 * (lane & 1) : 0);
                const bf16x8 f = fp4x8<__bf16>(code, e8m0_to_f32(p.vs[v * (DP / 32) + lane * NE / 32]));
#pragma unroll
                for (int e = 0; e < NE; ++e) acc[e] = __builtin_fmaf(wt, (float)f[e], acc[e]);
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
        if (x.splits > 1) {
            const int64_t at = ((int64_t)(b * a.kv_heads + hkv) * x.splits + share) * rows + row;
#pragma unroll
            for (int e = 0; e < NE; ++e) x.part[at * DP + lane * NE + e] = acc[e];
            if (lane == 0) x.part_m[at * 2] = m, x.part_m[at * 2 + 1] = l;
            continue;
        }
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
        for (int e = 0; e < NE; ++e) ((T *)a.o)[b * a.o_b + tok * a.o_t + h * a.o_h + lane * NE + e] = (T)(acc[e] * inv);
        if (a.lse && lane == 0)
            a.lse[b * a.lse_b + h * a.lse_h + tok] = l > 0.f ? m * a.c - kLift<T> + __log2f(l) : l != l ? l : -INFINITY;
    }
}

// Rows (tokens x heads of a key head) up to which each wave of the cache
// attention has them all; more run in tiles of 64, 16 a wave.  With 64 rows: 27
// us in tiles, 34 in blocks of 32 (8 x 4096 tokens of 4 key heads of 128), 20 and 17
// for one such sequence; with 32 the tiles are mostly padding.
constexpr int kDecodeRows = 32;
// The number of the first tile (as find_tile counts them) of sequence s.
LSMX_DEV int first_tile(const AttnArgs &a, const Seq &s, int size, int mult) {
    if (!a.offsets) return s.b * ((a.q_len * mult + size - 1) / size);
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int first = 0; first <= s.idx; first += 64) {
        const int i = first + lane;
        if (i < s.idx) {
            const int lo = i == 0 ? 0 : min(max(a.offsets[i - 1], 0), a.tokens), hi = min(max(a.offsets[i], 0), a.tokens);
            n += (int)(((int64_t)max(hi - lo, 0) * mult + size - 1) / size);
        }
    }
    for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
    return uniform(n);
}

hipError_t launch_kv_append(const AppendArgs &a, int dtype, hipStream_t s);
int kv_attend_splits(int batch, int kv_heads, int rows, int64_t keys);
hipError_t launch_kv_attend(const AttendArgs &a, int dtype, hipStream_t s);
hipError_t launch_kv_chunk(const AttendArgs &a, int dtype, hipStream_t s);
hipError_t launch_kv_weights(const AttendArgs &a, int dtype, hipStream_t s);
hipError_t launch_kv_evict(const EvictArgs &a, hipStream_t s);

hipError_t launch_attn_fwd(const AttnArgs &a, int dtype, hipStream_t s);
int64_t attn_bwd_workspace(const AttnArgs &a);
hipError_t launch_attn_bwd(const AttnArgs &a, int dtype, hipStream_t s);

}  // namespace lsmx
