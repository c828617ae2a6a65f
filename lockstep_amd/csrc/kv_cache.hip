// A paged MXFP4 key-value cache: writing it, attention over it for few rows,
// the accumulated weight of each key, and eviction.
#include "lsmx_attn.h"
#include "lsmx_q16.h"

namespace lsmx {
namespace {

// ------------------------------------------------------------------ append
// Four lanes quantize a 32-block (8 elements of 16 bits each); the rule and
// the bytes are those of the quantizer (lsmx_q16.h).
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
            *(bf16x8 *)out = fp4x8_to_bf16(codes, e8m0_to_f32(e8));
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
        const int hi = (len + 31) / 32;
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
    LSMX_DEV void load(const uint8_t *codes, const uint8_t *scale, int64_t v, int g, bool in) {
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = 0;
        e = 0;
        if (in) {
            const uint8_t *c = codes + v * (DP / 2) + g * (DP / 8);
            if constexpr (NW == 4)
                *(u32x4 *)w = *(const u32x4 *)c;
            else
                *(u32x2 *)w = *(const u32x2 *)c;
            e = scale[v * (DP / 32) + g * (DP / 32) / 4];
        }
    }
};

// Rows of one (sequence, key head): row -> token and head, q fragments whose
// contraction runs over quarter g of the vector in lane group g.
template <typename TQ, int DP, int NT>
LSMX_DEV void load_rows(const AttnArgs &a, int b, int hkv, int row, int g, bool in, bf16x8 (&q)[NT][DP / 32]) {
    typedef typename Vec<TQ>::x8 Q8;
    const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
    const TQ *qp = (const TQ *)a.q + b * a.q_b + tok * a.q_t + h * a.q_h + g * (DP / 4);
#pragma unroll
    for (int x = 0; x < DP / 32; ++x) {
        const Q8 w = in ? *(const Q8 *)(qp + x * 8) : Q8{};
        if constexpr (NT == 1)
            q[0][x] = w;
        else
            split(w, q[0][x], q[1][x]);
    }
}

// One workgroup: one sequence and key head, RT x 16 rows, a share of the keys;
// its 4 waves take tiles of 32 keys in turn and are joined at the end.
template <typename TQ, int DP, int RT>
__global__ __launch_bounds__(256) void kv_decode_kernel(AttendArgs x) {
    constexpr int NC = DP / 8, NS = DP / 32, ND = DP / 16, NT = __is_same(TQ, __bf16) ? 1 : 2;
    __shared__ __attribute__((aligned(16))) uint8_t smem[4 * 32 * DP * 2];  // values of a wave's tile; then 16 x DP fp32 of a wave
    __shared__ float s_m[4][16], s_l[4][16];
    const AttnArgs &a = x.a;
    const Pool &p = x.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int bh = blockIdx.x / x.splits, sp = blockIdx.x - bh * x.splits, b = bh / a.kv_heads, hkv = bh - b * a.kv_heads;
    const int rows = a.q_len * a.group;
    const Tiles tiles(x, b);
    const int i0 = (int)((int64_t)tiles.n * sp / x.splits), i1 = (int)((int64_t)tiles.n * (sp + 1) / x.splits);

    bf16x8 q[RT][NT][NS];
    int pos[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int row = t * 16 + r;
        load_rows<TQ, DP, NT>(a, b, hkv, row, g, row < rows, q[t]);
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
    __bf16 *sv = (__bf16 *)smem + wave * 32 * DP;
    const int pfirst = tiles.len - a.q_len;

    for (int i = i0 + wave; i < i1; i += 4) {
        const int j0 = tiles[i] * 32;
        Codes<DP> k[2], v[2];
        bool in[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int j = j0 + t * 16 + r, pg = j < tiles.len ? p.page_of(b, j) : -1;
            in[t] = pg >= 0;
            const int64_t vec = p.vec(max(pg, 0), hkv, j);
            k[t].load(p.kc, p.ks, vec, g, in[t]);
            v[t].load(p.vc, p.vs, vec, g, in[t]);
        }
        f32x4 st[2][RT];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const float ksc = e8m0_to_f32(k[t].e), vsc = e8m0_to_f32(v[t].e);
#pragma unroll
            for (int y = 0; y < RT; ++y) st[t][y] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const bf16x8 kf = fp4x8_to_bf16(k[t].w[s], ksc);
#pragma unroll
                for (int y = 0; y < RT; ++y)
#pragma unroll
                    for (int n = 0; n < NT; ++n) st[t][y] = mfma(kf, q[y][n][s], st[t][y]);
                const int row = t * 16 + r, c = g * NS + s;
                *(bf16x8 *)(sv + row * DP + swz<NC>(row, c) * 8) = fp4x8_to_bf16(v[t].w[s], vsc);
            }
        }
        // hidden keys: past a row's position, outside its window, or in no page
        const bool full = j0 + 31 <= pfirst && __all(in[0] & in[1]) && (!a.window || j0 > tiles.len - 1 - a.window || j0 + 31 < a.sinks);
        if (!full) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint64_t ok = __ballot(in[t]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int j = j0 + t * 16 + g * 4 + e;
                    const bool held = (ok >> (g * 4 + e)) & 1;
#pragma unroll
                    for (int y = 0; y < RT; ++y)
                        st[t][y][e] = (held & sees(j, pos[y], window_low(pos[y], a.window), a.sinks)) ? st[t][y][e] : -INFINITY;
                }
            }
        }
        bf16x8 pf[RT][NT];
#pragma unroll
        for (int y = 0; y < RT; ++y) {
            float mx = m[y];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, st[t][y][e]);
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float mc = mx == -INFINITY ? 0.f : mx * a.c;
            const float alpha = __builtin_amdgcn_exp2f(m[y] * a.c - mc);
            m[y] = mx;
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(st[t][y][e], a.c, -mc));
                    sum += w;
                    pf[y][0][t * 4 + e] = (__bf16)w;
                    if constexpr (NT == 2) pf[y][1][t * 4 + e] = (__bf16)(w - (float)pf[y][0][t * 4 + e]);
                }
            l[y] = l[y] * alpha + sum;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d][y] *= alpha;
        }
        // the wave's own LDS region: its writes above, its reads here
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        const int row = g * 4 + (r >> 2);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const int c = d * 2 + ((r & 3) >> 1), e = (r & 1) * 4;
            const bf16x8 vf = join<bf16x4, bf16x8>(read_tr<__bf16>(sv + row * DP + swz<NC>(row, c) * 8 + e),
                                                   read_tr<__bf16>(sv + (row + 16) * DP + swz<NC>(row + 16, c) * 8 + e));
#pragma unroll
            for (int y = 0; y < RT; ++y)
#pragma unroll
                for (int n = 0; n < NT; ++n) o[d][y] = mfma(vf, pf[y][n], o[d][y]);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    }

    // join the waves, 16 rows at a time
    float *so = (float *)smem;  // [4][16][DP] would not fit: halves of the head
    constexpr int HD = DP / 2;
#pragma unroll
    for (int y = 0; y < RT; ++y) {
        float sum = l[y] + __shfl_xor(l[y], 16);
        sum += __shfl_xor(sum, 32);
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
                    TQ *op = (TQ *)a.o + b * a.o_b + tok * a.o_t + h * a.o_h + half * HD + c;
                    const float inv = tot > 0.f || tot != tot ? 1.f / tot : 0.f;
#pragma unroll
                    for (int e = 0; e < HD / 16; ++e) op[e] = (TQ)(acc[e] * inv);
                    if (a.lse && half == 0 && (threadIdx.x & 15) == 0)
                        a.lse[b * a.lse_b + h * a.lse_h + tok] = tot > 0.f ? mc + __log2f(tot) : tot != tot ? tot : -INFINITY;
                }
            }
        }
    }
}

// Joins the shares of one row: one wave per row.
template <typename TQ, int DP>
__global__ __launch_bounds__(64) void kv_join_kernel(AttendArgs x) {
    const AttnArgs &a = x.a;
    const int rows = a.q_len * a.group, lane = threadIdx.x;
    const int row = blockIdx.x % rows, bh = blockIdx.x / rows, b = bh / a.kv_heads, hkv = bh - b * a.kv_heads;
    const int64_t at0 = (int64_t)bh * x.splits * rows + row;
    float top = -INFINITY;
    for (int s = lane; s < x.splits; s += 64) top = fmaxf(top, x.part_m[(at0 + (int64_t)s * rows) * 2]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float mc = top == -INFINITY ? 0.f : top * a.c;
    float tot = 0.f, acc[DP / 64];
#pragma unroll
    for (int e = 0; e < DP / 64; ++e) acc[e] = 0.f;
    for (int s = 0; s < x.splits; ++s) {
        const int64_t at = at0 + (int64_t)s * rows;
        const float f = __builtin_amdgcn_exp2f(x.part_m[at * 2] * a.c - mc);
        tot += x.part_m[at * 2 + 1] * f;
#pragma unroll
        for (int e = 0; e < DP / 64; ++e) acc[e] += x.part[at * DP + lane * (DP / 64) + e] * f;
    }
    const int tok = div_by(row, a.by_group), h = hkv * a.group + row - tok * a.group;
    TQ *op = (TQ *)a.o + b * a.o_b + tok * a.o_t + h * a.o_h + lane * (DP / 64);
    const float inv = tot > 0.f || tot != tot ? 1.f / tot : 0.f;
#pragma unroll
    for (int e = 0; e < DP / 64; ++e) op[e] = (TQ)(acc[e] * inv);
    if (a.lse && lane == 0)
        a.lse[b * a.lse_b + h * a.lse_h + tok] = tot > 0.f ? mc + __log2f(tot) : tot != tot ? tot : -INFINITY;
}

// ------------------------------------------------------------------ weights
// weights[b, h, j] += sum over the rows of exp(s_ij - lse_i), the scores
// recomputed from the keys' codes.  A wave owns 16 keys and runs over the rows
// in tiles of 16: one owner and one order for every sum.
template <typename TQ, int DP>
__global__ __launch_bounds__(256) void kv_weights_kernel(AttendArgs x) {
    constexpr int NS = DP / 32, NT = __is_same(TQ, __bf16) ? 1 : 2;
    const AttnArgs &a = x.a;
    const Pool &p = x.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int per = ((p.max_pages << p.page_shift) + 63) / 64;
    const int bh = blockIdx.x / per, b = bh / a.kv_heads, hkv = bh - b * a.kv_heads;
    const int len = p.length(b), rows = a.q_len * a.group, first = len - a.q_len;
    const int j0 = ((blockIdx.x - bh * per) * 4 + wave) * 16;
    if (j0 >= len) return;
    const int j = j0 + r, pg = j < len ? p.page_of(b, j) : -1;
    Codes<DP> k;
    k.load(p.kc, p.ks, p.vec(max(pg, 0), hkv, j), g, pg >= 0);
    const uint64_t ok = __ballot(pg >= 0);
    bf16x8 kf[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) kf[s] = fp4x8_to_bf16(k.w[s], e8m0_to_f32(k.e));
    // the rows that see some key of the tile
    const int tok_lo = max(0, j0 - first);
    int tok_hi = a.q_len;
    if (a.window && j0 >= a.sinks) tok_hi = min(tok_hi, min(j0 + 15, len - 1) + a.window - first);
    if (tok_lo >= tok_hi) return;
    f32x4 sum{0, 0, 0, 0};
    for (int r0 = tok_lo * a.group; r0 < tok_hi * a.group; r0 += 16) {
        const int row = r0 + r;
        const bool in = row < rows;
        bf16x8 q[NT][NS];
        load_rows<TQ, DP, NT>(a, b, hkv, row, g, in, q);
        const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
        const int pos = in ? tok + first : -1;
        const float lse = a.lse[b * a.lse_b + h * a.lse_h + tok];
        f32x4 st{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int n = 0; n < NT; ++n) st = mfma(kf[s], q[n][s], st);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool see = sees(j0 + g * 4 + e, pos, window_low(pos, a.window), a.sinks);
            sum[e] += see ? __builtin_amdgcn_exp2f(__builtin_fmaf(st[e], a.c, -lse)) : 0.f;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) sum[e] += __shfl_xor(sum[e], d);
        const int at = j0 + g * 4 + e;
        if (r == e && at < len && ((ok >> (g * 4 + e)) & 1)) x.weights[(int64_t)bh * x.w_len + at] += sum[e];
    }
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
// ascending order.
constexpr int kSelect = 1024;
__global__ __launch_bounds__(kSelect) void kv_select_kernel(EvictArgs a) {
    __shared__ int hist[256], s_scan[2][kSelect / 64], s_pick[2];
    const int bh = blockIdx.x, b = bh / a.p.kv_heads, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = a.p.length(b);
    const float *w = a.weights + (int64_t)bh * a.w_len;
    int32_t *index = a.index + (int64_t)bh * a.keep;
    float *kept = a.new_weights + (int64_t)bh * a.keep;
    if (bh % a.p.kv_heads == 0 && tid == 0) a.new_lengths[b] = min(n, a.keep);
    const int c0 = min(a.sinks, n), c1 = max(c0, n - a.recent);  // candidates
    const bool all = n <= a.keep;
    int want = all ? 0 : a.keep - (n - (c1 - c0));  // of the candidates
    uint32_t prefix = 0;
    if (!all) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int j = c0 + tid; j < c1; j += kSelect) {
                const uint32_t u = rank_of(w[j]);
                if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(u >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int left = want, bin = 255;
                while (bin > 0 && hist[bin] < left) left -= hist[bin--];
                s_pick[0] = bin, s_pick[1] = left;
            }
            __syncthreads();
            prefix |= (uint32_t)s_pick[0] << shift;
            want = s_pick[1];
            __syncthreads();
        }
    }
    // prefix is the rank of the last that stays, `want` the number of its
    // equals that do (the first of them)
    int ties = 0, out = 0;
    for (int j0 = 0; j0 < n; j0 += kSelect) {
        const int j = j0 + tid;
        const float x = j < n ? w[j] : 0.f;
        const uint32_t u = rank_of(x);
        const bool held = j < n && (all || j < c0 || j >= c1 || u > prefix);
        const bool tie = j < n && !all && j >= c0 && j < c1 && u == prefix;
        const uint64_t bt = __ballot(tie);
        if (lane == 0) s_scan[0][wave] = __popcll(bt);
        __syncthreads();
        int before = ties, all_ties = 0;
        for (int i = 0; i < kSelect / 64; ++i) {
            before += i < wave ? s_scan[0][i] : 0;
            all_ties += s_scan[0][i];
        }
        before += __popcll(bt & ((1ull << lane) - 1));
        const bool stay = held | (tie & (before < want));
        const uint64_t bs = __ballot(stay);
        if (lane == 0) s_scan[1][wave] = __popcll(bs);
        __syncthreads();
        int at = out, all_out = 0;
        for (int i = 0; i < kSelect / 64; ++i) {
            at += i < wave ? s_scan[1][i] : 0;
            all_out += s_scan[1][i];
        }
        at += __popcll(bs & ((1ull << lane) - 1));
        if (stay) index[at] = j, kept[at] = x;
        ties += all_ties;
        out += all_out;
        __syncthreads();
    }
    for (int i = out + tid; i < a.keep; i += kSelect) index[i] = -1, kept[i] = 0.f;
}

// Moves the kept vectors to the new pages: 16 threads per token's key and
// value vectors.
__global__ __launch_bounds__(256) void kv_move_kernel(EvictArgs a) {
    const Pool &p = a.p;
    const int per = (a.keep + 15) / 16;
    const int bh = blockIdx.x / per, b = bh / p.kv_heads, h = bh - b * p.kv_heads;
    const int to = (blockIdx.x - bh * per) * 16 + (threadIdx.x >> 4), c = threadIdx.x & 15;
    if (to >= min(a.keep, a.out_max_pages << p.page_shift)) return;
    const int from = a.index[(int64_t)bh * a.keep + to];
    if (from < 0) return;
    const int sp = p.page_of(b, from), dp = a.out_table[(int64_t)b * a.out_max_pages + (to >> p.page_shift)];
    if (sp < 0 || (uint32_t)dp >= (uint32_t)p.pages) return;
    const int64_t sv = p.vec(sp, h, from), dv = p.vec(dp, h, to);
    const int words = p.dim / 8;  // of codes; scales: dim / 32 bytes
    if (c < words) {
        ((uint32_t *)p.kc)[dv * words + c] = ((const uint32_t *)p.kc)[sv * words + c];
        ((uint32_t *)p.vc)[dv * words + c] = ((const uint32_t *)p.vc)[sv * words + c];
    }
    if (c < p.dim / 32) {
        p.ks[dv * (p.dim / 32) + c] = p.ks[sv * (p.dim / 32) + c];
        p.vs[dv * (p.dim / 32) + c] = p.vs[sv * (p.dim / 32) + c];
    }
}

template <typename TQ, int DP>
hipError_t attend(const AttendArgs &x, hipStream_t s) {
    const int rows = x.a.q_len * x.a.group, bh = x.a.batch * x.a.kv_heads;
    const dim3 grid((unsigned)x.splits * bh);
    if (rows <= 16)
        kv_decode_kernel<TQ, DP, 1><<<grid, 256, 0, s>>>(x);
    else if (rows <= 32)
        kv_decode_kernel<TQ, DP, 2><<<grid, 256, 0, s>>>(x);
    else
        kv_decode_kernel<TQ, DP, 4><<<grid, 256, 0, s>>>(x);
    if (x.splits > 1) kv_join_kernel<TQ, DP><<<(unsigned)(rows * bh), 64, 0, s>>>(x);
    return hipGetLastError();
}

template <typename TQ, int DP>
hipError_t weights(const AttendArgs &x, hipStream_t s) {
    const int keys = x.p.max_pages << x.p.page_shift;
    const dim3 grid((unsigned)((keys + 63) / 64) * x.a.batch * x.a.kv_heads);
    kv_weights_kernel<TQ, DP><<<grid, 256, 0, s>>>(x);
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
// keys (2 tiles per wave).
int kv_attend_splits(int batch, int kv_heads, int rows, int64_t keys) {
    if (rows > kDecodeRows) return 1;
    const int64_t bh = (int64_t)batch * kv_heads;
    const int64_t by_cu = (1024 + bh - 1) / bh, by_len = (keys + 255) / 256;
    const int64_t n = by_cu < by_len ? by_cu : by_len;
    return (int)(n < 1 ? 1 : n > 256 ? 256 : n);
}


hipError_t launch_kv_attend(const AttendArgs &x, int dtype, hipStream_t s) {
    if (x.a.q_len * x.a.group > kDecodeRows) return launch_kv_chunk(x, dtype, s);
    if (dtype == LSMX_BF16) return x.p.dim == 64 ? attend<__bf16, 64>(x, s) : attend<__bf16, 128>(x, s);
    return x.p.dim == 64 ? attend<_Float16, 64>(x, s) : attend<_Float16, 128>(x, s);
}

hipError_t launch_kv_weights(const AttendArgs &x, int dtype, hipStream_t s) {
    if (dtype == LSMX_BF16) return x.p.dim == 64 ? weights<__bf16, 64>(x, s) : weights<__bf16, 128>(x, s);
    return x.p.dim == 64 ? weights<_Float16, 64>(x, s) : weights<_Float16, 128>(x, s);
}

hipError_t launch_kv_evict(const EvictArgs &a, hipStream_t s) {
    const int bh = a.batch * a.p.kv_heads;
    kv_select_kernel<<<(unsigned)bh, kSelect, 0, s>>>(a);
    kv_move_kernel<<<(unsigned)((a.keep + 15) / 16) * bh, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace lsmx
