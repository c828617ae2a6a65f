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
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
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
// (8 or 16).  The 16 rows that one operand read touches fall on 16 different
// 16-byte bank groups, and so do the 8 rows x 2 chunks of half a transposing
// read.
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

// Workgroup id -> work item so that consecutive items stay on one of the 8
// XCDs (ids go to them in turn) and share its L2.  The grid is padded to a
// multiple of 8; items past `total` are dropped by the caller.
LSMX_DEV int xcd_item(int id, int per) { return (id & 7) * per + (id >> 3); }

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
    int tiles, per;  // tiles per kv head over all sequences (dense: of one sequence times batch); items per XCD
    // backward
    const void *d_o;
    int64_t do_b, do_t, do_h;
    float *delta;
    void *dq, *dk, *dv;  // contiguous, laid out as q, k, v
    float scale;
    float *part;         // partial gradients of the sink keys
    int sink_tiles, splits;
};

// One sequence of a packed or dense batch.
struct Seq {
    int b, q_len, k_len, shift;  // query token t has position t + shift
    int64_t q0, k0;              // first token (packed: in the token axis, else 0)
    int tile;
};

// The sequence and tile of work tile t, tiles of `size` rows with `mult` rows
// per token, `len` tokens in a dense sequence.  Packed tokens before offsets[0] and from offsets[batch] on
// belong to two more sequences that see nothing (k_len 0).
// Returns false past the last tile.
LSMX_DEV bool find_tile(const AttnArgs &a, int t, int size, int mult, int len, Seq &s) {
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
            s.tile = t - before - (__shfl(upto, w) - __shfl(n, w));
            s.q_len = __shfl(own, w);
            s.q0 = s.k0 = __shfl(lo, w);
            const int idx = first + w;
            s.b = 0;
            s.k_len = idx >= 1 && idx <= a.batch ? s.q_len : 0;
            s.shift = s.k_len ? 0 : -s.q_len;  // dead sequence: positions below 0
            return true;
        }
        before += __shfl(upto, 63);
    }
    return false;
}

hipError_t launch_attn_fwd(const AttnArgs &a, int dtype, hipStream_t s);
int64_t attn_bwd_workspace(const AttnArgs &a);
hipError_t launch_attn_bwd(const AttnArgs &a, int dtype, hipStream_t s);

}  // namespace lsmx
