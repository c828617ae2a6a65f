// A paged MXFP4 key-value cache: writing it, attention over it for few rows,
// the accumulated weight of each key, and eviction.
#include "lsmx_attn.h"
#include "lsmx_q16.h"

namespace lsmx {
namespace {

// ------------------------------------------------------------------ append
// Four lanes quantize a 32-block (8 elements of 16 bits each); the rule and
// the bytes are those of the quantizer (lsmx_q16.h).  A workgroup takes 512
// blocks' parts of k and v, so that few new tokens still spread over the chip.
// Bound by the bytes: 12000 tokens of 8 heads of 128, 25.5 us = 4.3 TB/s; 64 tokens,
// a launch's own 4.6 us.
constexpr int kAppendTokens = 64;  // most tokens of a workgroup

template <typename T>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a, int per_wg) {
    __shared__ int64_t s_vec[kAppendTokens];  // vector index of head 0, or -1
    const Pool &p = a.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t0 = blockIdx.x * per_wg, n = min(per_wg, a.tokens - t0);
    for (int i = wave; i < n; i += 4) {
        const int t = t0 + i;
        int b, left;  // sequence, tokens of it from t on
        if (a.offsets) {
            int count = 0;
            for (int f = 0; f <= a.batch; f += 64)
                count += __popcll(__ballot(f + lane <= a.batch && a.offsets[min(f + lane, a.batch)] <= t));
            b = count - 1;
            left = b >= 0 && b < a.batch ? min(a.offsets[b + 1], a.tokens) - t : 0;
        } else {
            b = div_by(t, a.by_seq);
            left = (b + 1) * a.per_seq - t;
        }
        if (lane == 0) {
            int64_t v = -1;
            if (left > 0) {
                const int len = p.lengths[b], j = len - left;
                if (j >= 0 && j < p.max_pages << p.page_shift) {
                    const int pg = p.page_of(b, j);
                    if (pg >= 0) v = p.vec(pg, 0, j);
                }
            }
            s_vec[i] = v;
        }
    }
    __syncthreads();
    const int cpv = p.dim / 8, per_tok = p.kv_heads * cpv;  // 8-element chunks
    for (int id = threadIdx.x; id < n * per_tok * 2; id += 256) {
        const bool is_v = id >= n * per_tok;
        const int x = is_v ? id - n * per_tok : id;
        const int i = x / per_tok, y = x - i * per_tok, h = y / cpv, c = y - h * cpv;
        const T *src = is_v ? (const T *)a.v + (int64_t)(t0 + i) * a.v_t + h * a.v_h
                            : (const T *)a.k + (int64_t)(t0 + i) * a.k_t + h * a.k_h;
        const u32x4 w = *(const u32x4 *)(src + c * 8);
        float f[8];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint16_t half = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            const uint32_t bits = f2u((float)__builtin_bit_cast(T, half));
            f[e] = nudge_keep_nan(bits);
            top = max(top, bits & 0x7FFFFFFFu);
        }
        top = max(top, (uint32_t)__shfl_xor((int)top, 1));
        top = max(top, (uint32_t)__shfl_xor((int)top, 2));
        const uint32_t e8 = block_e8m0_16x(top), codes = codes8_any(f, e8);
        const int64_t v0 = s_vec[i];
        if (v0 >= 0) {
            const int64_t v = v0 + ((int64_t)h << p.page_shift);
            *(uint32_t *)((is_v ? p.vc : p.kc) + v * (p.dim / 2) + c * 4) = codes;
            if ((c & 3) == 0) (is_v ? p.vs : p.ks)[v * (p.dim / 32) + (c >> 2)] = (uint8_t)e8;
        }
        if (a.k_out) {
            __bf16 *out = (__bf16 *)(is_v ? a.v_out : a.k_out) + ((int64_t)(t0 + i) * p.kv_heads + h) * p.dim + c * 8;
            *(bf16x8 *)out = fp4x8<__bf16>(codes, e8m0_to_f32(e8));
        }
    }
}

// ------------------------------------------------------------------ decode
// The tiles of 32 keys that the rows of a sequence see: the sinks' tiles,
// then those of the window.
struct Tiles {
    int sink, lo, n, len;
    LSMX_DEV Tiles(const AttendArgs &x, int b) {
        len = x.p.length(b);
        const int first = len - x.a.q_len;  // position of the first row
        const int hi = x.p.pages ? (len + 31) / 32 : 0;
        sink = min(hi, (x.a.sinks + 31) / 32);
        lo = x.a.window ? max(sink, max(0, first - x.a.window + 1) / 32) : sink;
        n = sink + max(0, hi - lo);
    }
    LSMX_DEV int operator[](int i) const { return i < sink ? i : lo + i - sink; }
};

// The codes of 16 keys: lane 16g + r holds the quarter g of the vector of key r.
template <int DP>
struct Codes {
    static constexpr int NW = DP / 32;
    uint32_t w[NW];
    uint32_t e;
    // codes, scale: of the first key (the same for the whole wave)
    LSMX_DEV void load(const uint8_t *codes, const uint8_t *scale, int g, int r) {
        const uint8_t *c = codes + r * (DP / 2) + g * (DP / 8);
        if constexpr (NW == 4)
            *(u32x4 *)w = *(const u32x4 *)c;
        else
            *(u32x2 *)w = *(const u32x2 *)c;
        e = scale[r * (DP / 32) + g * (DP / 32) / 4];
    }
    LSMX_DEV void drop() {
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = 0;
        e = 127;
    }
};

// 32 keys of a sequence and key head from position j0 on: two groups of 16,
// each within one page.  Every slot of a page can be read, so that the loads
// stand outside all branches; what lies in no page is read from the pool's
// first one, and hidden.
template <int DP, bool VALUES>
struct Keys {
    int j0, pg[2];  // pages, or -1
    Codes<DP> k[2], v[2];
    LSMX_DEV void load(const Pool &p, int h, int g, int r) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int64_t vec = p.vec(max(pg[t], 0), h, j0 + t * 16);
            k[t].load(p.kc + vec * (DP / 2), p.ks + vec * (DP / 32), g, r);
            if constexpr (VALUES) v[t].load(p.vc + vec * (DP / 2), p.vs + vec * (DP / 32), g, r);
        }
    }
};

// The tiles i0 + wave, i0 + wave + 4, .. of one wave, and their pages: 64 page
// numbers at a time, one of each lane, so that a tile's pages are at hand
// without a load of their own.
struct Walk {
    const Pool &p;
    const Tiles &tiles;
    int b, end, first, pages;  // first: the tile whose pages lanes 0 and 1 hold
    LSMX_DEV Walk(const Pool &pool, const Tiles &t, int seq, int i, int i1) : p(pool), tiles(t), b(seq), end(i1) { fill(i); }
    LSMX_DEV void fill(int i) {
        const int lane = threadIdx.x & 63, mine = i + 4 * (lane >> 1), j = tiles[mine] * 32 + (lane & 1) * 16;
        first = i;
        pages = mine < end && j < tiles.len ? p.page_of(b, j) : -1;
    }
    template <typename K>
    LSMX_DEV void find(int i, K &keys) {
        if (i - first >= 128) fill(i);
        const int at = (i - first) >> 1;
        keys.j0 = tiles[i] * 32;
        keys.pg[0] = lane_of(pages, at);
        keys.pg[1] = lane_of(pages, at + 1);
    }
};

// Rows of one (sequence, key head): row -> token and head, q fragments whose
// contraction runs over quarter g of the vector in lane group g.
template <typename T, int DP>
LSMX_DEV void load_rows(const AttnArgs &a, int b, int hkv, int row, int g, bool in, typename Vec<T>::x8 (&q)[DP / 32]) {
    typedef typename Vec<T>::x8 X8;
    const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
    const T *qp = (const T *)a.q + b * a.q_b + tok * a.q_t + h * a.q_h + g * (DP / 4);
#pragma unroll
    for (int x = 0; x < DP / 32; ++x) q[x] = in ? *(const X8 *)(qp + x * 8) : X8{};
}

// The scores of 16 keys, lane 16g + r holding keys 4g..4g+3 of row r (ROWS: rows
// 4g..4g+3 of key r); the lane's part of each vector is contracted as it lies in
// memory.
template <typename T, int DP, int RT, bool ROWS = false>
LSMX_DEV void scores(const Codes<DP> &k, const typename Vec<T>::x8 (&q)[RT][DP / 32], f32x4 (&st)[RT]) {
    // (the branches of the general form keep the operands of two groups of keys from
    // being made at once, which costs a wave per SIMD where registers are few)
    const float sc = ROWS || RT > 1 ? e8m0_to_f32(k.e) : block_scale<T>(k.e);
#pragma unroll
    for (int y = 0; y < RT; ++y) st[y] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < DP / 32; ++s) {
        const typename Vec<T>::x8 kf = fp4x8<T>(k.w[s], sc);
#pragma unroll
        for (int y = 0; y < RT; ++y) st[y] = ROWS ? mfma(q[y][s], kf, st[y]) : mfma(kf, q[y][s], st[y]);
    }
}

// One workgroup: one sequence and key head, its up to RT x 16 rows, a share of the keys;
// its 4 waves take tiles of 32 keys in turn and are joined at the end.  A wave
// has the next tile's codes in flight while it works on one, and the page
// numbers of the tile after that.
//
// Bound by the loads in flight, so that waves per SIMD count: 4 of them at 64 x
// 8192 tokens of 8 key heads of 128 take 82 us = 5.2 TB/s (3: 91, 2: 101).
template <typename T, int DP, int RT>
__global__ __launch_bounds__(256, RT > 1 && DP == 128 ? 2 : 4) void kv_decode_kernel(AttendArgs x) {
    constexpr int NC = DP / 8, NS = DP / 32, ND = DP / 16;
    typedef typename Vec<T>::x8 X8;
    typedef typename Vec<T>::x4 X4;
    __shared__ __attribute__((aligned(16))) uint8_t smem[4 * 32 * DP * 2];  // values of a wave's tile; then 16 x DP / 2 fp32 of a wave
    __shared__ float s_m[4][16], s_l[4][16];
    const AttnArgs &a = x.a;
    const Pool &p = x.p;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, r = lane & 15;
    const int rows = a.q_len * a.group;
    const int bh = blockIdx.x / x.splits, sp = blockIdx.x - bh * x.splits, b = bh / a.kv_heads, hkv = bh - b * a.kv_heads;
    const Tiles tiles(x, b);
    const int i0 = (int)((int64_t)tiles.n * sp / x.splits), i1 = (int)((int64_t)tiles.n * (sp + 1) / x.splits);

    Keys<DP, true> cur, nxt;
    int i = i0 + wave;
    Walk walk(p, tiles, b, i, i1);
    if (i < i1) {
        walk.find(i, cur);
        cur.load(p, hkv, g, r);
    }
    X8 q[RT][NS];
    int pos[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int row = t * 16 + r;
        load_rows<T, DP>(a, b, hkv, row, g, row < rows, q[t]);
        pos[t] = row < rows ? div_by(row, a.by_group) + tiles.len - a.q_len : -1;
    }
    f32x4 o[ND][RT];
    float m[RT], l[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        m[t] = -INFINITY, l[t] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d][t] = f32x4{0, 0, 0, 0};
    }
    T *sv = (T *)smem + wave * 32 * DP;
    const int pfirst = tiles.len - a.q_len;
    uint64_t bad = 0;  // lanes with a block that T does not hold

    for (; i < i1; i += 4) {
        // after the last tile this one again, from the cache: the loads of all
        // rounds are alike, and the wait is for the round before
        walk.find(i + 4 < i1 ? i + 4 : i, nxt);
        nxt.load(p, hkv, g, r);
        const int j0 = cur.j0;
        // the lane's places in LDS, made anew each round: held over the loop they
        // would take the registers of a wave
        int lr = r;
        asm volatile("" : "+v"(lr));
        // hidden keys: past a row's position, outside its window, or in no page
        const bool full = j0 + 31 <= pfirst && (cur.pg[0] | cur.pg[1]) >= 0 &&
                          (!a.window || j0 > tiles.len - 1 - a.window || j0 + 31 < a.sinks);
        if (!full) {
            // what is in no row's sight must not reach a product as a NaN
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (cur.pg[t] < 0 || j0 + t * 16 + r >= tiles.len) {
                    cur.v[t].drop();
                    if constexpr (__is_same(T, _Float16)) cur.k[t].e = 127;
                }
        }
        f32x4 st[2][RT];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            bad |= __ballot(!(holds<T>(cur.k[t].e) & holds<T>(cur.v[t].e)));
            scores<T, DP, RT>(cur.k[t], q, st[t]);
            const float vsc = RT > 1 ? e8m0_to_f32(cur.v[t].e) : block_scale<T>(cur.v[t].e);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const int row = t * 16 + lr, c = g * NS + s;
                *(X8 *)(sv + row * DP + swz<NC>(row, c) * 8) = fp4x8<T>(cur.v[t].w[s], vsc);
            }
        }
        if (!full) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = j0 + t * 16 + g * 4 + e;
#pragma unroll
                    for (int y = 0; y < RT; ++y) {
                        const bool see = (cur.pg[t] >= 0) & sees(j, pos[y], window_low(pos[y], a.window), a.sinks);
                        st[t][y][e] = see ? st[t][y][e] : -INFINITY;
                    }
                }
        }
        X8 pf[RT];
#pragma unroll
        for (int y = 0; y < RT; ++y) {
            float mx = st[0][y][0];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, st[t][y][e]);
            if (__any(mx > m[y])) {
                const float top = fmaxf(m[y], max_rows(mx));
                const float alpha = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[y] - top) * a.c);
                m[y] = top;
                l[y] *= alpha;
#pragma unroll
                for (int d = 0; d < ND; ++d) o[d][y] *= alpha;
            }
            const float mc = m[y] == -INFINITY ? 0.f : m[y] * a.c - kLift<T>;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(st[t][y][e], a.c, -mc));
                    l[y] += w;
                    pf[y][t * 4 + e] = (T)w;
                }
        }
        // the wave's own LDS region: its writes above, its reads here, in order
        asm volatile("" ::: "memory");
        const int row = g * 4 + (lr >> 2);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const int c = d * 2 + ((lr & 3) >> 1), e = (lr & 1) * 4;
            const X8 vf = join<X4, X8>(read_tr<T>(sv + row * DP + swz<NC>(row, c) * 8 + e),
                                                   read_tr<T>(sv + (row + 16) * DP + swz<NC>(row + 16, c) * 8 + e));
#pragma unroll
            for (int y = 0; y < RT; ++y) o[d][y] = mfma(vf, pf[y], o[d][y]);
        }
        asm volatile("" ::: "memory");
        cur = nxt;
    }
    if constexpr (__is_same(T, _Float16)) {
        if (uniform(__syncthreads_or(bad != 0))) {
            attend_exact<T, DP, 32>(x, b, hkv, sp, 0, rows, i1 - i0, [=](int k) { return tiles[i0 + k] * 32; });
            return;
        }
    }

    // join the waves, 16 rows at a time
    float *so = (float *)smem;  // [4][16][DP] would not fit: halves of the head
    constexpr int HD = DP / 2;
#pragma unroll
    for (int y = 0; y < RT; ++y) {
        const float sum = sum_rows(l[y]);
        __syncthreads();
        if (g == 0) s_m[wave][r] = m[y], s_l[wave][r] = sum;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            __syncthreads();
#pragma unroll
            for (int d = 0; d < ND / 2; ++d)
                *(f32x4 *)(so + (wave * 16 + r) * HD + d * 16 + g * 4) = o[half * (ND / 2) + d][y];
            __syncthreads();
            const int row = threadIdx.x >> 4, c = (threadIdx.x & 15) * (HD / 16), full = y * 16 + row;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, s_m[w][row]);
            const float mc = top == -INFINITY ? 0.f : top * a.c;
            float tot = 0.f, acc[HD / 16];
#pragma unroll
            for (int e = 0; e < HD / 16; ++e) acc[e] = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = __builtin_amdgcn_exp2f(s_m[w][row] * a.c - mc);
                tot += s_l[w][row] * f;
#pragma unroll
                for (int e = 0; e < HD / 16; ++e) acc[e] += so[(w * 16 + row) * HD + c + e] * f;
            }
            if (full < rows) {
                if (x.splits > 1) {
                    const int64_t at = ((int64_t)bh * x.splits + sp) * rows + full;
#pragma unroll
                    for (int e = 0; e < HD / 16; ++e) x.part[at * DP + half * HD + c + e] = acc[e];
                    if (half == 0 && (threadIdx.x & 15) == 0) x.part_m[at * 2] = top, x.part_m[at * 2 + 1] = tot;
                } else {
                    const int tok = div_by(full, a.by_group), h = hkv * a.group + full - tok * a.group;
                    T *op = (T *)a.o + b * a.o_b + tok * a.o_t + h * a.o_h + half * HD + c;
                    const float inv = tot > 0.f || tot != tot ? 1.f / tot : 0.f;
#pragma unroll
                    for (int e = 0; e < HD / 16; ++e) op[e] = (T)(acc[e] * inv);
                    if (a.lse && half == 0 && (threadIdx.x & 15) == 0)
                        a.lse[b * a.lse_b + h * a.lse_h + tok] = tot > 0.f ? mc - kLift<T> + __log2f(tot) : tot != tot ? tot : -INFINITY;
                }
            }
        }
    }
}

// Joins up to 16 shares of a row: 16 threads over the vector, 16 rows a
// workgroup.  Bound by the shares' bytes: 19200 rows of 3 shares of 64, 5.6 us.
template <typename T, int DP>
__global__ __launch_bounds__(256) void kv_join_few_kernel(AttendArgs x) {
    constexpr int NE = DP / 16;
    const AttnArgs &a = x.a;
    const int rows = a.q_len * a.group, c = (threadIdx.x & 15) * NE;
    const int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (i >= (int64_t)rows * a.batch * a.kv_heads) return;
    const int bh = (int)(i / rows), row = (int)(i - (int64_t)bh * rows), b = bh / a.kv_heads, hkv = bh - b * a.kv_heads;
    const int64_t at0 = (int64_t)bh * x.splits * rows + row;
    float top = -INFINITY;
    for (int s = 0; s < x.splits; ++s) top = fmaxf(top, x.part_m[(at0 + (int64_t)s * rows) * 2]);
    const float mc = top == -INFINITY ? 0.f : top * a.c;
    float tot = 0.f, acc[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int s = 0; s < x.splits; ++s) {
        const int64_t at = at0 + (int64_t)s * rows;
        const float f = __builtin_amdgcn_exp2f(x.part_m[at * 2] * a.c - mc);
        tot = __builtin_fmaf(x.part_m[at * 2 + 1], f, tot);
#pragma unroll
        for (int e = 0; e < NE; e += 4) {
            const f32x4 w = *(const f32x4 *)(x.part + at * DP + c + e);
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[e + k] = __builtin_fmaf(w[k], f, acc[e + k]);
        }
    }
    const int tok = div_by(row, a.by_group), h = hkv * a.group + row - tok * a.group;
    const float inv = tot > 0.f || tot != tot ? 1.f / tot : 0.f;
    T *o = (T *)a.o + b * a.o_b + tok * a.o_t + h * a.o_h + c;
#pragma unroll
    for (int e = 0; e < NE; e += 4)
        *(typename Vec<T>::x4 *)(o + e) = typename Vec<T>::x4{(T)(acc[e] * inv), (T)(acc[e + 1] * inv), (T)(acc[e + 2] * inv), (T)(acc[e + 3] * inv)};
    if (a.lse && c == 0)
        a.lse[b * a.lse_b + h * a.lse_h + tok] = tot > 0.f ? mc - kLift<T> + __log2f(tot) : tot != tot ? tot : -INFINITY;
}

// Joins the shares of one row: 16 threads over the vector, 16 over the shares;
// for one long sequence, whose shares are many and rows few (32 rows of 128
// shares of 128: 4.2 us, a launch and two dependent loads).
template <typename T, int DP>
__global__ __launch_bounds__(256) void kv_join_kernel(AttendArgs x) {
    constexpr int NE = DP / 16;
    __shared__ float s_top[4], s_tot[16], s_acc[16][DP + 4];
    const AttnArgs &a = x.a;
    const int rows = a.q_len * a.group, lane = threadIdx.x & 63, part = threadIdx.x >> 4, c = (threadIdx.x & 15) * NE;
    const int row = blockIdx.x % rows, bh = blockIdx.x / rows, b = bh / a.kv_heads, hkv = bh - b * a.kv_heads;
    const int64_t at0 = (int64_t)bh * x.splits * rows + row;
    float top = -INFINITY;
    for (int s = threadIdx.x; s < x.splits; s += 256) top = fmaxf(top, x.part_m[(at0 + (int64_t)s * rows) * 2]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (lane == 0) s_top[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    const float mc = top == -INFINITY ? 0.f : top * a.c;
    float tot = 0.f, acc[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int s = part; s < x.splits; s += 16) {
        const int64_t at = at0 + (int64_t)s * rows;
        const float f = __builtin_amdgcn_exp2f(x.part_m[at * 2] * a.c - mc);
        tot = __builtin_fmaf(x.part_m[at * 2 + 1], f, tot);
#pragma unroll
        for (int e = 0; e < NE; e += 4) {
            const f32x4 w = *(const f32x4 *)(x.part + at * DP + c + e);
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[e + k] = __builtin_fmaf(w[k], f, acc[e + k]);
        }
    }
#pragma unroll
    for (int e = 0; e < NE; ++e) s_acc[part][c + e] = acc[e];
    if (c == 0) s_tot[part] = tot;
    __syncthreads();
    if (threadIdx.x >= DP) return;
    float sum = 0.f;
    tot = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += s_acc[i][threadIdx.x], tot += s_tot[i];
    const int tok = div_by(row, a.by_group), h = hkv * a.group + row - tok * a.group;
    const float inv = tot > 0.f || tot != tot ? 1.f / tot : 0.f;
    ((T *)a.o)[b * a.o_b + tok * a.o_t + h * a.o_h + threadIdx.x] = (T)(sum * inv);
    if (a.lse && threadIdx.x == 0)
        a.lse[b * a.lse_b + h * a.lse_h + tok] = tot > 0.f ? mc - kLift<T> + __log2f(tot) : tot != tot ? tot : -INFINITY;
}

// ------------------------------------------------------------------ weights
// weights[b, h, j] += sum over the rows of exp(s_ij - lse_i), the scores
// recomputed from the keys' codes.  Each sum has one owner and one order.
// (Scores kept by the first pass are fewer bytes for up to 8 rows at head 128,
// but their short runs made that pass 118 us from 80 at 64 x 8192 tokens of 8
// key heads and 4 rows, and adding them took 42, where this takes 47.)
//
// Few rows: the q of RT x 16 stays in registers, and the waves run over the keys
// as in kv_decode_kernel, once for each such block.  Bound by the codes' bytes:
// 64 sequences of up to 8192 tokens of 8 key heads of 128, 4 rows each, 47 us =
// 5.0 TB/s.
LSMX_DEV float sum_16(float x) {  // over the 16 lanes of a row of lanes
    x += u2f(__builtin_amdgcn_update_dpp(0, f2u(x), 0xB1, 0xF, 0xF, true));   // quad_perm 1,0,3,2
    x += u2f(__builtin_amdgcn_update_dpp(0, f2u(x), 0x4E, 0xF, 0xF, true));   // quad_perm 2,3,0,1
    x += u2f(__builtin_amdgcn_update_dpp(0, f2u(x), 0x141, 0xF, 0xF, true));  // row_half_mirror
    x += u2f(__builtin_amdgcn_update_dpp(0, f2u(x), 0x140, 0xF, 0xF, true));  // row_mirror
    return x;
}
// The weight of key j, vector vec, over every step-th row of [row0, row1), in fp32
// (holds).
template <typename T, int DP>
LSMX_DEV float weight_exact(const AttendArgs &x, int b, int hkv, int j, int64_t vec, int row0, int row1, int step) {
    const AttnArgs &a = x.a;
    const int shift = x.p.length(b) - a.q_len;
    float sum = 0.f;
#pragma unroll 1
    for (int row = row0; row < row1; row += step) {
        const int tok = div_by(row, a.by_group), h = hkv * a.group + row - tok * a.group;
        const T *q = (const T *)a.q + b * a.q_b + tok * a.q_t + h * a.q_h;
        const float s = dot_exact(q, x.p.kc + vec * (DP / 2), x.p.ks + vec * (DP / 32), DP);
        const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(s, a.c, -a.lse[b * a.lse_b + h * a.lse_h + tok]));
        sum += sees(j, tok + shift, window_low(tok + shift, a.window), a.sinks) ? v : 0.f;
    }
    return sum;
}
// Whether T holds the blocks of a tile's keys before position len.
template <typename T, int DP>
LSMX_DEV bool all_held(const Keys<DP, false> &k, int len) {
    if constexpr (!__is_same(T, _Float16)) return true;
    const int r = threadIdx.x & 15;
    return __all((holds<T>(k.k[0].e) | (k.j0 + r >= len)) & (holds<T>(k.k[1].e) | (k.j0 + 16 + r >= len)));
}
// The weights over the tiles i, i + 4, .. that it does not hold.
template <typename T, int DP>
LSMX_DEV void weights_exact(const AttendArgs &x, int b, int hkv, int i, int i1) {
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));  // as in attend_exact
    const Pool &p = x.p;
    const int lane = thread & 63, g = lane >> 4, r = lane & 15;
    const Tiles tiles(x, b);
    Walk walk(p, tiles, b, i, i1);
    Keys<DP, false> cur;
    for (; i < i1; i += 4) {
        walk.find(i, cur);
        cur.load(p, hkv, g, r);
        const int j = cur.j0 + (lane & 31), pg = g == 0 ? cur.pg[0] : cur.pg[1];
        if (!all_held<T, DP>(cur, tiles.len) && lane < 32 && j < tiles.len && pg >= 0)
            x.weights[(int64_t)(b * x.a.kv_heads + hkv) * x.w_len + j] +=
                weight_exact<T, DP>(x, b, hkv, j, p.vec(pg, hkv, j), 0, x.a.q_len * x.a.group, 1);
    }
}
template <typename T, int DP, int RT>
__global__ __launch_bounds__(256) void kv_weights_kernel(AttendArgs x) {
    constexpr int NS = DP / 32;
    typedef typename Vec<T>::x8 X8;
    const AttnArgs &a = x.a;
    const Pool &p = x.p;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, r = lane & 15;
    const int bh = blockIdx.x / x.splits, sp = blockIdx.x - bh * x.splits, b = bh / a.kv_heads, hkv = bh - b * a.kv_heads;
    const int rows = a.q_len * a.group;
    const Tiles tiles(x, b);
    const int i0 = (int)((int64_t)tiles.n * sp / x.splits), i1 = (int)((int64_t)tiles.n * (sp + 1) / x.splits);
    if (i0 + wave >= i1) return;
    float *w = x.weights + (int64_t)bh * x.w_len;
    bool left = false;
    for (int row0 = 0; row0 < rows; row0 += RT * 16) {
        Keys<DP, false> cur, nxt;
        int i = i0 + wave;
        Walk walk(p, tiles, b, i, i1);
        walk.find(i, cur);
        cur.load(p, hkv, g, r);
        X8 q[RT][NS];
        int pos[RT][4];
        float lse[RT][4];  // of rows 4g..4g+3; past the last: infinite, a weight of 0
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            load_rows<T, DP>(a, b, hkv, row0 + t * 16 + r, g, row0 + t * 16 + r < rows, q[t]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = row0 + t * 16 + g * 4 + e;
                const bool in = row < rows;
                const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
                pos[t][e] = in ? tok + tiles.len - a.q_len : -1;
                lse[t][e] = in ? a.lse[b * a.lse_b + h * a.lse_h + tok] : INFINITY;
            }
        }
        const int pfirst = div_by(row0, a.by_group) + tiles.len - a.q_len;
        for (; i < i1; i += 4) {
            const int j0 = cur.j0;
            // the first 32 lanes keep the sums of a key each
            const int mine = j0 + (lane & 31);
            const bool held = lane < 32 && mine < tiles.len && (g == 0 ? cur.pg[0] : cur.pg[1]) >= 0;
            float before = held ? w[mine] : 0.f;
            // after the last tile this one again, from the cache: the loads of all
            // rounds are alike, and the wait is for the round before
            walk.find(i + 4 < i1 ? i + 4 : i, nxt);
            nxt.load(p, hkv, g, r);
            const bool full = j0 + 31 <= pfirst && (!a.window || j0 > tiles.len - 1 - a.window || j0 + 31 < a.sinks);
            const bool ok = all_held<T, DP>(cur, full ? 0x7FFFFFFF : tiles.len);
            left = left | !ok;
            float sum[2] = {0.f, 0.f};
            auto add = [&](auto all) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    f32x4 st[RT];  // rows 4g..4g+3 of key r
                    scores<T, DP, RT, true>(cur.k[t], q, st);
#pragma unroll
                    for (int y = 0; y < RT; ++y)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(st[y][e], a.c, -lse[y][e]));
                            if constexpr (decltype(all)::value)
                                sum[t] += v;
                            else
                                sum[t] += sees(j0 + t * 16 + r, pos[y][e], window_low(pos[y][e], a.window), a.sinks) ? v : 0.f;
                        }
                }
            };
            if (full)
                add(BoolC<true>{});
            else
                add(BoolC<false>{});
            const float s0 = sum_rows(sum[0]), s1 = sum_rows(sum[1]);
            if (held & ok) w[mine] = before + (g == 0 ? s0 : s1);
            cur = nxt;
        }
    }
    if (left) weights_exact<T, DP>(x, b, hkv, i0 + wave, i1);
}

// Many rows: a workgroup owns 64 keys, whose operands stay in registers, and
// its waves take tiles of 16 rows in turn; their sums are joined in LDS.  Bound
// by the loads of q in flight and, below some 500 workgroups, by their number:
// 12 waves each then, else 4.  16/4 heads, T newest tokens of B sequences, us:
//     head 64:  T = 600, B = 2, window 2048 (340 at work)  4 waves 35, 8: 34, 12: 31
//               T = 600, B = 2 of 5000 (632)               4 waves 32, 8: 44, 12: 40
//     head 128: T = 20, B = 8 of 4096 (2048)               4 waves 18, 8: 45, 12: 39
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64) void kv_weights_rows_kernel(AttendArgs x) {
    constexpr int NS = DP / 32;
    __shared__ __attribute__((aligned(16))) float s_sum[NW][64];
    typedef typename Vec<T>::x8 X8;
    const AttnArgs &a = x.a;
    const Pool &p = x.p;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, r = lane & 15;
    const int per = ((p.max_pages << p.page_shift) + 63) / 64;
    const int bh = blockIdx.x / per, b = bh / a.kv_heads, hkv = bh - b * a.kv_heads;
    const int len = p.length(b), first = len - a.q_len, j0 = (blockIdx.x - bh * per) * 64;
    if (j0 >= len) return;
    // the rows that see some key of the tile
    const int tok_lo = max(0, j0 - first);
    int tok_hi = a.q_len;
    if (a.window && j0 >= a.sinks) tok_hi = min(tok_hi, min(j0 + 63, len - 1) + a.window - first);
    if (tok_lo >= tok_hi) return;
    X8 kf[4][NS];
    int pg[4];
    bool ok = true;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int j = j0 + t * 16;
        pg[t] = uniform(j < len ? p.page_of(b, j) : -1);
        const int64_t vec = p.vec(max(pg[t], 0), hkv, j);
        Codes<DP> k;
        if (p.pages)
            k.load(p.kc + vec * (DP / 2), p.ks + vec * (DP / 32), g, r);
        else
            k.drop();
#pragma unroll
        for (int s = 0; s < NS; ++s) kf[t][s] = fp4x8<T>(k.w[s], block_scale<T>(k.e));
        ok = ok && (holds<T>(k.e) || pg[t] < 0 || j + r >= len);
    }
    auto put = [&] {  // the waves' sums of the 64 keys
        __syncthreads();
        const int at = j0 + threadIdx.x;
        if (threadIdx.x < 64 && at < len) {
            float all = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) all += s_sum[i][threadIdx.x];
            x.weights[(int64_t)bh * x.w_len + at] += all;
        }
    };
    if constexpr (__is_same(T, _Float16)) {
        if (!__all(ok)) {  // in every wave alike
            const int j = j0 + lane, own = j < len ? p.page_of(b, j) : -1;
            s_sum[wave][lane] = own < 0 ? 0.f : weight_exact<T, DP>(x, b, hkv, j, p.vec(own, hkv, j), tok_lo * a.group + wave, tok_hi * a.group, NW);
            put();
            return;
        }
    }
    f32x4 sum[4];
    uint32_t span[4][4];  // position p sees key j when 0 <= p - j <= span
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        sum[t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) span[t][e] = a.window && j0 + t * 16 + g * 4 + e >= a.sinks ? a.window - 1 : 0x7FFFFFFF;
    }
    const int row_hi = tok_hi * a.group;
    // U tiles of rows at a time, the next U in flight: one tile's work is less
    // than a load's latency
    constexpr int U = 128 / DP, kStep = NW * 16;
    struct Row {
        X8 q[NS];
        float lse;
        int pos;
    };
    auto load = [&](int r0, Row (&w)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int row = r0 + u * kStep + r;
            const bool in = row < row_hi;
            const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
            const T *qp = (const T *)a.q + b * a.q_b + tok * a.q_t + h * a.q_h + g * (DP / 4);
#pragma unroll
            for (int s = 0; s < NS; ++s) w[u].q[s] = *(const X8 *)(qp + s * 8);
            w[u].lse = a.lse[b * a.lse_b + h * a.lse_h + tok];
            w[u].pos = in ? tok + first : -1;
        }
    };
    Row cur[U], nxt[U];
    int r0 = tok_lo * a.group + wave * 16;
    load(r0, cur);
    for (; r0 < row_hi; r0 += kStep * U) {
        load(r0 + kStep * U, nxt);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            auto add = [&](auto all) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    f32x4 st{0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < NS; ++s) st = mfma(kf[t][s], cur[u].q[s], st);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(st[e], a.c, -cur[u].lse));
                        if constexpr (decltype(all)::value)
                            sum[t][e] += v;
                        else
                            sum[t][e] += (uint32_t)(cur[u].pos - (j0 + t * 16 + g * 4 + e)) <= span[t][e] ? v : 0.f;
                    }
                }
            };
            // every row sees every key: most tiles
            if (__all(cur[u].pos >= j0 + 63 && (!a.window || cur[u].pos < j0 + a.window || j0 + 63 < a.sinks)))
                add(BoolC<true>{});
            else
                add(BoolC<false>{});
            cur[u] = nxt[u];
        }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float all = sum_16(sum[t][e]);
            if (r == 0) s_sum[wave][t * 16 + g * 4 + e] = pg[t] >= 0 ? all : 0.f;
        }
    put();
}

// ------------------------------------------------------------------ eviction
// Bits whose unsigned order is the order of the weights: -0 equals 0, a NaN is
// above all.
LSMX_DEV uint32_t rank_of(float w) {
    const uint32_t b = f2u(w + 0.f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
    return b >> 31 ? ~b : b | 0x80000000u;
}

// One workgroup per sequence and key head: the rank of the last weight that
// stays, by radix selection 8 bits at a time, then the kept positions in
// ascending order.  Bound by the four rounds' own latency (histogram in LDS, a
// search of its bins): 256 x 8192 weights 16 us, 8 x 1500 8 us.
// PER: ranks a thread keeps in registers, which covers
// 1024 PER positions; 0: they are read again in each round.
constexpr int kSelect = 1024;
template <int PER>
__global__ __launch_bounds__(kSelect) void kv_select_kernel(EvictArgs a) {
    __shared__ int hist[256], s_scan[2][kSelect / 64], s_lost[kSelect / 64], s_pick[2];
    const int bh = blockIdx.x, b = bh / a.p.kv_heads, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = a.p.length(b);
    const float *w = a.weights + (int64_t)bh * a.w_len;
    int32_t *index = a.index + (int64_t)bh * a.keep;
    float *kept = a.new_weights + (int64_t)bh * a.keep;
    const int c0 = min(a.sinks, n), c1 = max(c0, n - a.recent);  // candidates
    uint32_t prefix = 0, there = ~0u;  // bit k: of round k
    float own[PER ? PER : 1];
#pragma unroll
    for (int k = 0; k < PER; ++k) own[k] = k * kSelect + tid < n ? w[k * kSelect + tid] : 0.f;
    // positions in no page are not there
    bool lost = false;
    for (int g = tid; g << a.p.page_shift < n; g += kSelect) lost = lost | (a.p.page_of(b, g << a.p.page_shift) < 0);
    const bool any = __any(lost);
    if (lane == 0) s_lost[wave] = any;
    __syncthreads();
    const bool holes = __any(s_lost[lane % (kSelect / 64)]);
    if (PER > 0 && holes) {
        for (int k = 0; k < PER; ++k) {
            const int j = k * kSelect + tid;
            if (j < n && a.p.page_of(b, j) < 0) there &= ~(1u << k);
        }
    }
    // body(position, weight, whether it is there), by all threads alike
    auto each = [&](auto body) {
        if constexpr (PER > 0) {
#pragma unroll
            for (int k = 0; k < PER; ++k)
                if (k * kSelect < n) body(k * kSelect + tid, own[k], (there >> k) & 1);
        } else {
            if (holes) {
                for (int j = tid; j - tid < n; j += kSelect) body(j, j < n ? w[j] : 0.f, j < n && a.p.page_of(b, j) >= 0);
            } else {
                for (int j = tid; j - tid < n; j += kSelect) body(j, j < n ? w[j] : 0.f, true);
            }
        }
    };
    int total = n, free = c1 - c0;
    if (holes) {
        if (tid < 2) s_pick[tid] = 0;
        __syncthreads();
        int gone = 0, gone_free = 0;
        each([&](int j, float, bool in) {
            const bool no = j < n && !in;
            gone += no, gone_free += no && j >= c0 && j < c1;
        });
        atomicAdd(&s_pick[0], gone);
        atomicAdd(&s_pick[1], gone_free);
        __syncthreads();
        total -= s_pick[0], free -= s_pick[1];
        __syncthreads();
    }
    const bool all = total <= a.keep;
    int want = all ? 0 : a.keep - (total - free);  // of the candidates
    if (bh % a.p.kv_heads == 0 && tid == 0) a.new_lengths[b] = min(total, a.keep);
    if (!all) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            each([&](int j, float x, bool in) {
                const uint32_t u = rank_of(x);
                if (in && j >= c0 && j < c1 && (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))))
                    atomicAdd(&hist[(u >> shift) & 255], 1);
            });
            __syncthreads();
            if (wave == 0) {
                // the bin where the count from above reaches `want`: 4 bins a
                // lane, the topmost in lane 0
                int h[4], sum = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) sum += h[k] = hist[255 - (lane * 4 + k)];
                int above = sum;
                for (int d = 1; d < 64; d <<= 1) {
                    const int x = __shfl_up(above, d);
                    if (lane >= d) above += x;
                }
                const uint64_t reach = __ballot(above >= want);
                const int who = reach ? __ffsll((unsigned long long)reach) - 1 : 63;
                if (lane == who) {
                    int left = want - (above - sum), k = 0;
                    while (k < 3 && h[k] < left) left -= h[k++];
                    s_pick[0] = 255 - (lane * 4 + k), s_pick[1] = left;
                }
            }
            __syncthreads();
            prefix |= (uint32_t)s_pick[0] << shift;
            want = s_pick[1];
        }
    }
    // prefix is the rank of the last that stays, `want` the number of its
    // equals that do (the first of them)
    const uint64_t below = (1ull << lane) - 1;
    auto held = [&](int j, uint32_t u, bool in) { return in && j < n && (all || j < c0 || j >= c1 || u > prefix); };
    auto tie = [&](int j, uint32_t u, bool in) { return in && j < n && !all && j >= c0 && j < c1 && u == prefix; };
    int out = 0;
    if constexpr (PER > 0) {
        // counts of all (round, wave) pairs at once: their sums before each pair
        constexpr int NP = PER * (kSelect / 64), E = NP / 64;
        __shared__ int s_pair[NP + 1];
        auto scan = [&] {
            __syncthreads();
            if (wave == 0) {
                int v[E], sum = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) sum += v[e] = s_pair[lane * E + e];
                int upto = sum;
                for (int d = 1; d < 64; d <<= 1) {
                    const int x = __shfl_up(upto, d);
                    if (lane >= d) upto += x;
                }
                int at = upto - sum;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    s_pair[lane * E + e] = at;
                    at += v[e];
                }
                if (lane == 63) s_pair[NP] = at;
            }
            __syncthreads();
        };
        uint32_t stay = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const uint64_t m = __ballot(tie(k * kSelect + tid, rank_of(own[k]), (there >> k) & 1));
            if (lane == 0) s_pair[k * (kSelect / 64) + wave] = __popcll(m);
        }
        scan();
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int j = k * kSelect + tid;
            const uint32_t u = rank_of(own[k]);
            const bool t = tie(j, u, (there >> k) & 1);
            const uint64_t m = __ballot(t);
            const bool in = held(j, u, (there >> k) & 1) | (t & (s_pair[k * (kSelect / 64) + wave] + __popcll(m & below) < want));
            stay |= (uint32_t)in << k;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const uint64_t m = __ballot((stay >> k) & 1);
            if (lane == 0) s_pair[k * (kSelect / 64) + wave] = __popcll(m);
        }
        scan();
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const bool in = (stay >> k) & 1;
            const uint64_t m = __ballot(in);
            const int at = s_pair[k * (kSelect / 64) + wave] + __popcll(m & below);
            if (in) index[at] = k * kSelect + tid, kept[at] = own[k];
        }
        out = s_pair[NP];
    } else {
        int ties = 0;
        each([&](int j, float x, bool is) {
            const uint32_t u = rank_of(x);
            const bool t = tie(j, u, is);
            const uint64_t bt = __ballot(t);
            if (lane == 0) s_scan[0][wave] = __popcll(bt);
            __syncthreads();
            // sums over the waves before, and over all
            auto scan = [&](const int *v, int &before, int &total) {
                const int x = lane < kSelect / 64 ? v[lane] : 0;
                int y = lane < wave ? x : 0, z = x;
#pragma unroll
                for (int d = 1; d < kSelect / 64; d <<= 1) y += __shfl_xor(y, d), z += __shfl_xor(z, d);
                before = lane_of(y, 0), total = lane_of(z, 0);
            };
            int before, total;
            scan(s_scan[0], before, total);
            const bool in = held(j, u, is) | (t & (ties + before + __popcll(bt & below) < want));
            ties += total;
            const uint64_t bs = __ballot(in);
            if (lane == 0) s_scan[1][wave] = __popcll(bs);
            __syncthreads();
            scan(s_scan[1], before, total);
            const int at = out + before + __popcll(bs & below);
            if (in) index[at] = j, kept[at] = x;
            out += total;
        });
    }
    for (int i = out + tid; i < a.keep; i += kSelect) index[i] = -1, kept[i] = 0.f;
}

// Moves the kept vectors to the new pages: 8 threads a token, 4 for its key's
// codes and 4 for its value's; 4 tokens a thread, whose loads are in flight
// together.  Bound by the bytes, read in runs of single tokens: 32 x 8 heads of
// 4096 tokens of 128, 67 us = 4.3 TB/s.
template <int DP>
__global__ __launch_bounds__(256) void kv_move_kernel(EvictArgs a) {
    constexpr int NB = DP / 8, NW = NB / 4;  // bytes and words of codes of a thread
    typedef uint32_t Words __attribute__((ext_vector_type(NW)));
    const Pool &p = a.p;
    const int per = (a.keep + 127) / 128;
    const int bh = blockIdx.x / per, b = bh / p.kv_heads, h = bh - b * p.kv_heads;
    const int c = threadIdx.x & 3, is_v = (threadIdx.x >> 2) & 1, to0 = (blockIdx.x - bh * per) * 128 + (threadIdx.x >> 3);
    uint8_t *codes = is_v ? p.vc : p.kc, *scale = is_v ? p.vs : p.ks;
    int64_t src[4], dst[4];
    Words w[4];
    uint32_t e[4];
    int from[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int to = to0 + i * 32;
        from[i] = to < min(a.keep, a.out_max_pages << p.page_shift) ? a.index[(int64_t)bh * a.keep + to] : -1;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int to = to0 + i * 32;
        const int sp = from[i] >= 0 ? p.page_of(b, from[i]) : -1;
        const int dp = from[i] >= 0 ? a.out_table[(int64_t)b * a.out_max_pages + (to >> p.page_shift)] : -1;
        src[i] = sp >= 0 && (uint32_t)dp < (uint32_t)p.pages ? p.vec(sp, h, from[i]) : -1;
        dst[i] = p.vec(max(dp, 0), h, to);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (src[i] < 0) continue;
        w[i] = *(const Words *)(codes + src[i] * (DP / 2) + c * NB);
        if (c == 0) e[i] = DP == 128 ? *(const uint32_t *)(scale + src[i] * 4) : *(const uint16_t *)(scale + src[i] * 2);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (src[i] < 0) continue;
        *(Words *)(codes + dst[i] * (DP / 2) + c * NB) = w[i];
        if (c == 0) {
            if constexpr (DP == 128)
                *(uint32_t *)(scale + dst[i] * 4) = e[i];
            else
                *(uint16_t *)(scale + dst[i] * 2) = (uint16_t)e[i];
        }
    }
}

template <typename T, int DP>
hipError_t attend(const AttendArgs &x, hipStream_t s) {
    const int rows = x.a.q_len * x.a.group, bh = x.a.batch * x.a.kv_heads;
    const unsigned grid = (unsigned)x.splits * bh;
    if (rows <= 16)
        kv_decode_kernel<T, DP, 1><<<grid, 256, 0, s>>>(x);
    else
        kv_decode_kernel<T, DP, 2><<<grid, 256, 0, s>>>(x);
    return hipGetLastError();
}

template <typename T, int DP>
hipError_t join(const AttendArgs &x, hipStream_t s) {
    const int64_t rows = (int64_t)x.a.q_len * x.a.group * x.a.batch * x.a.kv_heads;
    if (x.splits > 16)
        kv_join_kernel<T, DP><<<(unsigned)rows, 256, 0, s>>>(x);
    else if (x.splits > 1)
        kv_join_few_kernel<T, DP><<<(unsigned)((rows + 15) / 16), 256, 0, s>>>(x);
    return hipGetLastError();
}

template <typename T, int DP>
hipError_t weights(AttendArgs x, hipStream_t s) {
    const int rows = x.a.q_len * x.a.group, bh = x.a.batch * x.a.kv_heads;
    const int64_t cap = (int64_t)x.p.max_pages << x.p.page_shift, reach = (int64_t)x.a.q_len + x.a.window + x.a.sinks;
    const int64_t keys = x.a.window && reach < cap ? reach : cap;
    // nothing is joined here: three times the shares of attention, for six waves per
    // SIMD, while each has 1024 keys (64 x 8192 tokens of 8 key heads of 128: 47 us
    // from 54; below, a share's start costs more: 64 x 2048 of 4 heads 12 from 10)
    const int least = kv_attend_splits(x.a.batch, x.a.kv_heads, 1, keys);
    x.splits = max(least, (int)min((int64_t)3 * least, keys / 1024));
    const unsigned grid = (unsigned)x.splits * bh;
    // up to 64 rows are one pass over the codes; up to three passes are still
    // faster than tiles of keys that each wait for the rows, where those would be
    // many.  64 x 2048 tokens of 4 key heads of 128: 24, 44, 64, 83 us for 64, 128,
    // 192, 256 rows, in tiles 60, 73, 83, 93; 8 x 4096 tokens: 10, 16, 24, 29 and 16, 20, 25,
    // 28; one sequence (64 tiles a head): 128 rows 12 and 6.
    const bool many = keys / 64 * bh >= 512;
    if (rows <= 16)
        kv_weights_kernel<T, DP, 1><<<grid, 256, 0, s>>>(x);
    else if (rows <= 32)
        kv_weights_kernel<T, DP, 2><<<grid, 256, 0, s>>>(x);
    else if (rows <= (many ? 192 : 64))
        kv_weights_kernel<T, DP, 4><<<grid, 256, 0, s>>>(x);
    else {
        const unsigned tiles = (unsigned)((cap + 63) / 64) * bh;
        if (many)
            kv_weights_rows_kernel<T, DP, 4><<<tiles, 256, 0, s>>>(x);
        else
            kv_weights_rows_kernel<T, DP, 12><<<tiles, 768, 0, s>>>(x);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_append(const AppendArgs &a, int dtype, hipStream_t s) {
    const int chunks = a.p.kv_heads * (a.p.dim / 8) * 2;
    const int per = chunks >= 512 ? 1 : (512 / chunks > kAppendTokens ? kAppendTokens : 512 / chunks);
    const unsigned grid = (unsigned)((a.tokens + per - 1) / per);
    if (dtype == LSMX_BF16)
        kv_append_kernel<__bf16><<<grid, 256, 0, s>>>(a, per);
    else
        kv_append_kernel<_Float16><<<grid, 256, 0, s>>>(a, per);
    return hipGetLastError();
}

// Shares of the keys: enough workgroups for 4 per CU, each of at least 256
// keys (2 tiles per wave).  A workgroup has all rows of a key head, or of many
// rows 64; there the shares' sums are most of the bytes, and no more than 16 are
// made (1.5 times as many workgroups: 37 + 7 us for 38 + 6, half: 43 + 5).
int kv_attend_splits(int batch, int kv_heads, int rows, int64_t keys) {
    const int64_t bh = (int64_t)batch * kv_heads, items = rows > kDecodeRows ? bh * ((rows + 63) / 64) : bh;
    const int64_t by_cu = rows > kDecodeRows ? (1024 + items / 2) / items : (1024 + items - 1) / items, by_len = (keys + 255) / 256;
    const int64_t n = by_cu < by_len ? by_cu : by_len, most = rows > kDecodeRows ? 16 : 256;
    return (int)(n < 1 ? 1 : n > most ? most : n);
}

hipError_t launch_kv_attend(const AttendArgs &x, int dtype, hipStream_t s) {
    const bool wide = x.p.dim == 128, bf16 = dtype == LSMX_BF16;
    const hipError_t e = x.a.q_len * x.a.group > kDecodeRows ? launch_kv_chunk(x, dtype, s)
                         : bf16                              ? (wide ? attend<__bf16, 128>(x, s) : attend<__bf16, 64>(x, s))
                                : (wide ? attend<_Float16, 128>(x, s) : attend<_Float16, 64>(x, s));
    if (e != hipSuccess) return e;
    return bf16 ? (wide ? join<__bf16, 128>(x, s) : join<__bf16, 64>(x, s))
                : (wide ? join<_Float16, 128>(x, s) : join<_Float16, 64>(x, s));
}

hipError_t launch_kv_weights(const AttendArgs &x, int dtype, hipStream_t s) {
    if (dtype == LSMX_BF16) return x.p.dim == 64 ? weights<__bf16, 64>(x, s) : weights<__bf16, 128>(x, s);
    return x.p.dim == 64 ? weights<_Float16, 64>(x, s) : weights<_Float16, 128>(x, s);
}

hipError_t launch_kv_evict(const EvictArgs &a, hipStream_t s) {
    const int bh = a.batch * a.p.kv_heads, cap = a.p.max_pages << a.p.page_shift;
    if (cap <= 4 * kSelect)
        kv_select_kernel<4><<<(unsigned)bh, kSelect, 0, s>>>(a);
    else if (cap <= 8 * kSelect)
        kv_select_kernel<8><<<(unsigned)bh, kSelect, 0, s>>>(a);
    else if (cap <= 32 * kSelect)
        kv_select_kernel<32><<<(unsigned)bh, kSelect, 0, s>>>(a);
    else
        kv_select_kernel<0><<<(unsigned)bh, kSelect, 0, s>>>(a);
    const unsigned grid = (unsigned)((a.keep + 127) / 128) * bh;
    if (a.p.dim == 64)
        kv_move_kernel<64><<<grid, 256, 0, s>>>(a);
    else
        kv_move_kernel<128><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace lsmx
