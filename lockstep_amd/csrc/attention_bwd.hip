// Attention with a sliding window and sinks: gradients.
//
//   P_ij = exp(s_ij - lse_i),  dV_j = sum_i P_ij dO_i,
//   dS_ij = P_ij (dO_i . v_j - delta_i),  delta_i = dO_i . o_i,
//   dQ_i = scale sum_j dS_ij k_j,  dK_j = scale sum_i dS_ij q_i.
//
// Two kernels, so that every sum has one order (no atomics): one owns rows and
// runs over their keys (dQ), the other owns keys and runs over the rows of all
// heads that share them (dK, dV).  Both recompute S and dP:
// eight products (dQ has dS in two terms) where one kernel with shared accumulators would
// take five, or six.
//
// The sinks are seen by every row: their keys would keep one workgroup busy
// with the whole sequence while the others have a window of it.  So the rows
// past the window of the sinks' tile are taken in chunks by a kernel of their
// own first, 16 sinks at a time, and the owner of the sinks adds the chunks'
// fp32 sums, in their order, before it rounds.
//
// Layouts as in the forward kernel: S^T = K Q^T feeds dQ^T += K^T dS^T without a
// lane crossing, and S = Q K^T feeds dV^T += dO^T P and dK^T += Q^T dS.
#include "lsmx_attn.h"
#include "lsmx_dma.h"

namespace lsmx {
namespace {

constexpr int kBN = 64;   // dQ: keys of a tile
constexpr int kKM = 128;  // dK, dV: keys of a workgroup
constexpr int kFar = 128; // far rows: rows of a tile

// fp16 holds 2^-24 to 65504, and gradients are often small: P enters its
// product times 2^10, and dS times a power of two of its own row (dQ) or key
// (dK) that is chosen when a value passes kTop and brings the largest so far
// to 2^10; the sums so far are rescaled, as the softmax does.  bf16 needs
// neither.
template <typename T>
struct Range {
    static constexpr bool on = __is_same(T, _Float16);
    static constexpr float kTop = 32768.f, kP = on ? 10.f : 0.f;
    // the power of two that brings x > 0 into [2^10, 2^11); 1 for inf and NaN,
    // and no more than 2^100
    LSMX_DEV static float scale_for(float x) {
        const int e = (int)((f2u(x) >> 23) & 255) - 127;
        return e >= 128 ? 1.f : __builtin_amdgcn_ldexpf(1.f, min(10 - e, 100));
    }
};

// 64 rows of one tensor straight into LDS, by the four waves of a workgroup;
// offset(row, chunk) is the byte offset in rs of 16-byte chunk `chunk`, or
// one past its end for zeros.
template <typename T, int DP, typename F>
LSMX_DEV void fetch_rows(v4i_rsrc rs, T *to, int rows, F offset) {
    constexpr int NC = DP / 8;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t lds = lds_u32(to);
#pragma unroll
    for (int u = 0; u < rows * NC / 256; ++u) {
        const int at = (u * 4 + wave) * 64, j = (at + lane) / NC, c = swz<NC>(j, lane % NC);
        dma_x4(offset(j, c), rs, lds + at * 16);
    }
}
constexpr uint32_t kZeros = 0x80000000u;

// Operand of 8 contraction rows 4g.., 16 + 4g.. of a tile from row j0 on, at
// columns 16 d + r.
template <typename T, int DP>
LSMX_DEV typename Vec<T>::x8 columns(const T *t, int j0, int d, int g, int r) {
    constexpr int NC = DP / 8;
    const int j = j0 + g * 4 + (r >> 2), c = d * 2 + ((r & 3) >> 1), e = (r & 1) * 4;
    return join<typename Vec<T>::x4, typename Vec<T>::x8>(read_tr<T>(t + j * DP + swz<NC>(j, c) * 8 + e),
                                                          read_tr<T>(t + (j + 16) * DP + swz<NC>(j + 16, c) * 8 + e));
}

// acc and the sum of x, two elements at a time.
LSMX_DEV float sum_of(bf16x8 x, float acc) {
    const bf16x2 one{(__bf16)1.f, (__bf16)1.f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) acc = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{x[i], x[i + 1]}, one, acc, false);
    return acc;
}

// ------------------------------------------------------------------ dQ, delta
// The dS of a row add up to 0, so that dQ_i = scale sum_j dS_ij (k_j - c_i) for any c_i.
// They do so up to what the forward's rounded probabilities left in o, hence in
// delta; with c_i near sum_j P_ij k_j, this residue r_i = sum_j dS_ij, kept in fp32, does
// not meet a common part of the keys: dQ_i = scale (sum_j dS_ij k_j - r_i c_i).  c_i takes
// the keys of the wave's last tile as they are (of its halves that some row sees: what is
// hidden from all may hold anything), with their P, and for the row's others their
// mean, as far as the row looks at keys in general: by its weight on the tile's
// keys, none counted above four times its share, against their share.  (A row that
// looks at one key takes nothing from others; one of few keys has most in the tile.)
// Keys with a common part of twice their spread: the error of dQ was 2.0 to 2.2 times
// that of rounding it, now 1.05; of four times 3.4, now 1.1 to 1.2.  Over 40000 random
// shapes, masks and scales no element takes more than 0.6 of its bound (each
// rounding's 4 u of its terms' magnitudes); without the cuts some passed it.
//
// Each workgroup owns 64 RT rows, a wave 16 RT: q and dO in registers, the keys through
// LDS as in the forward kernel.  delta comes first, from o and what o's rounding
// left out.  Bound as attn_dkv_kernel is (vector unit 63%, matrix unit 37%; two
// waves per SIMD): 2 x 4096 tokens, 32/8 heads of 128, window 1024: 354 us for
// four products (dS in two terms) = 682 TFLOP/s of the visible pairs.
template <typename T, int DP, int RT>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void attn_dq_kernel(AttnArgs a) {
    constexpr int NC = DP / 8, NS = DP / 32, ND = DP / 16, kBM = 64 * RT;
    // bf16 at head 128: dS is summed as it enters the products, two elements an
    // instruction, beside them (18 us where single additions before them took 25); fp16,
    // and head 64, the other way round (8 x 2048 tokens of 16/4 heads of 64, causal: 14 us of 650,
    // and 25)
    constexpr bool kSumLate = DP == 128 && !Range<T>::on;
    typedef typename Vec<T>::x8 X8;
    typedef typename Vec<T>::x4 X4;
    __shared__ __attribute__((aligned(16))) T sk[2][kBN * DP], sv[2][kBN * DP];

    const Item item = item_of(a, 1);
    const int hkv = item.head;
    if (hkv >= a.kv_heads) return;
    Seq s;
    if (!find_tile(a, a.tiles - 1 - item.tile, kBM, a.group, a.q_len, s)) return;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, r = lane & 15;
    const int row0 = s.tile * kBM, rows = s.q_len * a.group, wrow0 = row0 + wave * 16 * RT;

    const int pmin = div_by(row0, a.by_group) + s.shift;
    const int pmax = div_by(min(row0 + kBM, rows) - 1, a.by_group) + s.shift;
    const int hi = min(pmax + 1, s.k_len), lo = a.window ? max(0, pmin - a.window + 1) : 0;
    const int t_sink = (min(a.sinks, hi) + kBN - 1) / kBN, t_hi = hi > 0 ? (hi + kBN - 1) / kBN : 0;
    const int t_lo = lo / kBN;
    auto next = [&](int t) { return t + 1 < t_sink ? t + 1 : max(t + 1, t_lo); };
    int t = t_sink > 0 ? 0 : t_lo, n = 0;
    const int wmin = div_by(min(wrow0, rows - 1), a.by_group) + s.shift;
    const int wmax = wrow0 < rows ? div_by(min(wrow0 + 16 * RT, rows) - 1, a.by_group) + s.shift : -1;
    const int t_own = wmax >= 0 ? wmax / kBN : -1;  // the last tile that some row of the wave sees

    const T *kp = (const T *)a.k + s.b * a.k_b + s.k0 * a.k_t + hkv * a.k_h;
    const T *vp = (const T *)a.v + s.b * a.v_b + s.k0 * a.v_t + hkv * a.v_h;
    auto fetch = [&](int j0, int to) {
        const auto at = [&](int64_t x_t) {
            return [=](int j, int c) {
                return j0 + j < s.k_len && c * 8 < a.dim ? (uint32_t)(j * (int)x_t + c * 8) * 2 : kZeros;
            };
        };
        fetch_rows<T, DP>(buf_rsrc(kp + j0 * a.k_t, 0x7FFFFFFF), sk[to], kBN, at(a.k_t));
        fetch_rows<T, DP>(buf_rsrc(vp + j0 * a.v_t, 0x7FFFFFFF), sv[to], kBN, at(a.v_t));
    };
    if (t < t_hi) fetch(t * kBN, 0);

    int pos[RT], low[RT];
    float lse[RT], delta[RT], mul[RT] = {}, limit[RT] = {}, rest[RT] = {};  // rest: sum of dS over the lane's keys
    X8 qf[RT][NS], of[RT][NS];
#pragma unroll
    for (int y = 0; y < RT; ++y) {
        const int row = wrow0 + r + 16 * y;
        const bool in = row < rows;
        const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
        pos[y] = in ? tok + s.shift : -1;
        low[y] = window_low(pos[y], a.window);
        const int64_t l_at = s.b * a.lse_b + h * a.lse_h + s.q0 + tok;
        const T *qp = (const T *)a.q + s.b * a.q_b + (s.q0 + tok) * a.q_t + h * a.q_h;
        const T *dp = (const T *)a.d_o + s.b * a.do_b + (s.q0 + tok) * a.do_t + h * a.do_h;
        const int64_t o_at = s.b * a.o_b + (s.q0 + tok) * a.o_t + h * a.o_h;
        lse[y] = in ? a.lse[l_at] : 0.f;
        // delta from o as the forward had it: its rounded value and the rest
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < NS; ++x) {
            const int c = x * 4 + g;
            const bool ok = in && c * 8 < a.dim;
            qf[y][x] = ok ? *(const X8 *)(qp + c * 8) : X8{};
            of[y][x] = ok ? *(const X8 *)(dp + c * 8) : X8{};
            const X8 hi8 = ok ? *(const X8 *)((const T *)a.o + o_at + c * 8) : X8{};
            const X8 lo8 = ok ? *(const X8 *)((const T *)a.o_lo + o_at + c * 8) : X8{};
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = __builtin_fmaf((float)of[y][x][i], (float)hi8[i] + (float)lo8[i], sum);
        }
        delta[y] = sum_rows(sum);
        if (in && g == 0) a.delta[l_at] = delta[y];
    }
    f32x4 dq[ND][RT];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int y = 0; y < RT; ++y) dq[d][y] = f32x4{0, 0, 0, 0};

    wait_dma();
    __syncthreads();
    while (t < t_hi) {
        const int j0 = t * kBN, tn = next(t);
        if (tn < t_hi) fetch(tn * kBN, n ^ 1);
        const T *ck = sk[n], *cv = sv[n];
        // hidden from every row of the wave
        auto unseen = [&](int ju) { return ju > wmax || (a.window && ju + 31 <= wmin - a.window && ju >= a.sinks); };
        auto half = [&](auto all, int u) {
            const int ju = j0 + u * 32;
            // places in LDS made anew each time: held, they would not fit
            int lr = r;
            if constexpr (DP == 128) asm volatile("" : "+v"(lr));
            f32x4 st[2][RT], dp[2][RT];  // [16 keys][16 rows]
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const int j = u * 32 + w * 16 + lr;
#pragma unroll
                for (int y = 0; y < RT; ++y) st[w][y] = dp[w][y] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int x = 0; x < NS; ++x) {
                    const X8 kf = *(const X8 *)(ck + j * DP + swz<NC>(j, x * 4 + g) * 8);
                    const X8 vf = *(const X8 *)(cv + j * DP + swz<NC>(j, x * 4 + g) * 8);
#pragma unroll
                    for (int y = 0; y < RT; ++y) {
                        st[w][y] = mfma(kf, qf[y][x], st[w][y]);
                        dp[w][y] = mfma(vf, of[y][x], dp[w][y]);
                    }
                }
            }
            bool grow = false;
            float top[RT] = {};
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int y = 0; y < RT; ++y) {
                        float ds = __builtin_amdgcn_exp2f(__builtin_fmaf(st[w][y][i], a.c, -lse[y])) *
                                   (dp[w][y][i] - delta[y]);
                        if constexpr (!decltype(all)::value) {
                            const int j = ju + w * 16 + g * 4 + i;
                            ds = sees(j, pos[y], low[y], a.sinks) ? ds : 0.f;
                        }
                        st[w][y][i] = ds;
                        if constexpr (!kSumLate) rest[y] += ds;
                        if constexpr (Range<T>::on) top[y] = fmaxf(top[y], __builtin_fabsf(ds));
                    }
            if constexpr (Range<T>::on) {
                #pragma unroll
                for (int y = 0; y < RT; ++y) grow = grow | (top[y] > limit[y]);
                if (__any(grow)) {
#pragma unroll
                    for (int y = 0; y < RT; ++y) {
                        const float most = max_rows(top[y]);
                        if (most > limit[y]) {
                            const float m = Range<T>::scale_for(most), f = mul[y] == 0.f ? 0.f : m / mul[y];
                            mul[y] = m, limit[y] = Range<T>::kTop / m;
#pragma unroll
                            for (int d = 0; d < ND; ++d) dq[d][y] *= f;
                        }
                    }
                }
            }
            // two terms: the dS of a row cancel, so that with one rounding of each the
            // error of dQ is 1.4 times that of rounding it, and 2.5 times with keys that have a
            // common part of twice their spread; with two 1.01 and 1.05.  (60 us of 330.)
            X8 df[RT], dl[RT];
#pragma unroll
            for (int y = 0; y < RT; ++y)
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float ds = Range<T>::on ? st[w][y][i] * mul[y] : st[w][y][i];
                        df[y][w * 4 + i] = (T)ds;
                        dl[y][w * 4 + i] = (T)(ds - (float)df[y][w * 4 + i]);
                    }
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const X8 kf = columns<T, DP>(ck, u * 32, d, g, lr);
#pragma unroll
                for (int y = 0; y < RT; ++y) {
                    dq[d][y] = mfma(kf, df[y], dq[d][y]);
                    dq[d][y] = mfma(kf, dl[y], dq[d][y]);
                }
            }
            if constexpr (kSumLate) {
#pragma unroll
                for (int y = 0; y < RT; ++y) rest[y] = sum_of(df[y], sum_of(dl[y], rest[y]));
            }
        };
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int ju = j0 + u * 32;
            if (unseen(ju)) continue;
            if (ju + 31 <= wmin && (!a.window || ju > wmax - a.window || ju + 31 < a.sinks))
                half(BoolC<true>{}, u);
            else
                half(BoolC<false>{}, u);
        }
        if (t == t_own) {  // the rows' dS are complete: less r c (16 rows at a time: 32 do not fit)
#pragma unroll
            for (int y = 0; y < RT; ++y) {
                const int near = a.window ? min(pos[y] + 1, a.window) : pos[y] + 1;
                const float keys = (float)(near + min(a.sinks, pos[y] + 1 - near));  // that the row sees
                X8 pf[2];
                float mass = 0.f, even = 0.f, seen = 0.f, held = 0.f;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    pf[u] = X8{};
                    const int ju = j0 + u * 32;
                    if (unseen(ju)) continue;
                    held += (float)min(32, s.k_len - ju);
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        int lr = r;
                        asm volatile("" : "+v"(lr));  // as above
                        const int j = u * 32 + w * 16 + lr;
                        f32x4 st{0, 0, 0, 0};
#pragma unroll
                        for (int x = 0; x < NS; ++x)
                            st = mfma(*(const X8 *)(ck + j * DP + swz<NC>(j, x * 4 + g) * 8), qf[y][x], st);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i], a.c, -lse[y]));
                            const bool in = sees(ju + w * 16 + g * 4 + i, pos[y], low[y], a.sinks);
                            const float p = in ? e : 0.f;
                            mass += p;
                            even += fminf(p * keys, 4.f);
                            seen += in ? 1.f : 0.f;
                            pf[u][w * 4 + i] = (T)p;
                        }
                    }
                }
                const float sum = sum_rows(rest[y]) * (Range<T>::on ? mul[y] : 1.f);
                const float other = fmaxf(1.f - sum_rows(mass), 0.f) * fminf(1.f, 2.f * sum_rows(even) / (sum_rows(seen) + 8.f));
                const float each = keys >= 32.f ? other / held : 0.f;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (unseen(j0 + u * 32)) continue;
#pragma unroll
                    for (int i = 0; i < 8; ++i) pf[u][i] = (T)((float)pf[u][i] + each);
                    int lr = r;
                    asm volatile("" : "+v"(lr));
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        const f32x4 c = mfma(columns<T, DP>(ck, u * 32, d, g, lr), pf[u], f32x4{0, 0, 0, 0});
#pragma unroll
                        for (int i = 0; i < 4; ++i) dq[d][y][i] = __builtin_fmaf(-sum, c[i], dq[d][y][i]);
                    }
                }
            }
        }
        n ^= 1, t = tn;
        wait_dma();
        __syncthreads();
    }
#pragma unroll
    for (int y = 0; y < RT; ++y) {
        const int row = wrow0 + r + 16 * y;
        if (row >= rows) continue;
        const int tok = div_by(row, a.by_group), h = hkv * a.group + row - tok * a.group;
        T *p = (T *)a.dq + (((a.offsets ? s.q0 : (int64_t)s.b * a.q_len) + tok) * a.heads + h) * a.dim;
        const float f = !Range<T>::on ? a.scale : mul[y] == 0.f ? 0.f : a.scale / mul[y];
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            X4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (T)(dq[d][y][i] * f);
            if (d * 16 + g * 4 < a.dim) *(X4 *)(p + d * 16 + g * 4) = w;
        }
    }
}

// ------------------------------------------------------------------ dK, dV
// The rows of a (sequence, key head) from row0 on, gathered into LDS: q and dO,
// and each row's lse, delta and position.
template <typename T, int DP>
struct Rows {
    const AttnArgs &a;
    const Seq &s;
    int hkv, end;
    LSMX_DEV void fetch(int row0, T *sq, T *so, int count) {
        const int tok0 = uniform(div_by(row0, a.by_group)), last = end, dim = a.dim;
        const FastDiv by = a.by_group;
        auto at = [=](int64_t x_t, int64_t x_h) {
            return [=](int j, int c) {
                const int row = row0 + j, tok = div_by(row, by);
                return row < last && c * 8 < dim
                           ? (uint32_t)((tok - tok0) * (int)x_t + (row - tok * (int)by.d) * (int)x_h + c * 8) * 2
                           : kZeros;
            };
        };
        const T *q = (const T *)a.q + s.b * a.q_b + (s.q0 + tok0) * a.q_t + hkv * a.group * a.q_h;
        const T *d = (const T *)a.d_o + s.b * a.do_b + (s.q0 + tok0) * a.do_t + hkv * a.group * a.do_h;
        fetch_rows<T, DP>(buf_rsrc(q, 0x7FFFFFFF), sq, count, at(a.q_t, a.q_h));
        fetch_rows<T, DP>(buf_rsrc(d, 0x7FFFFFFF), so, count, at(a.do_t, a.do_h));
    }
    LSMX_DEV void stats(int row, float &lse, float &delta, int &pos) {
        const bool in = row < end;
        const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
        const int64_t at = s.b * a.lse_b + h * a.lse_h + s.q0 + tok;
        lse = in ? a.lse[at] - Range<T>::kP : 0.f;
        delta = in ? a.delta[at] : 0.f;
        pos = in ? tok + s.shift : -1;
    }
};

// 32 rows from row j0 of an LDS tile on against NK x 16 keys, whose K is in
// registers, and V too or (VL) in LDS.
template <typename T, int DP, int NK, bool VL>
struct KeySums {
    static constexpr int NC = DP / 8, NS = DP / 32, ND = DP / 16;
    typedef typename Vec<T>::x8 X8;
    X8 kf[NK][NS], vf[VL ? 1 : NK][NS];
    const T *sv;  // VL: the first key's row of V
    f32x4 dk[ND][NK], dv[ND][NK];
    float mul[NK], limit[NK];
    // position p sees key y of the lane when 0 <= p - key <= span
    int key[NK];
    uint32_t span[NK];

    LSMX_DEV void init(const AttnArgs &a, int key0) {
#pragma unroll
        for (int y = 0; y < NK; ++y) {
            key[y] = key0 + y * 16;
            span[y] = a.window && key[y] >= a.sinks ? a.window - 1 : 0x7FFFFFFF;
            mul[y] = limit[y] = 0.f;
#pragma unroll
            for (int d = 0; d < ND; ++d) dk[d][y] = dv[d][y] = f32x4{0, 0, 0, 0};
        }
    }
    LSMX_DEV void add(const T *sq, const T *so, const float *s_lse, const float *s_delta, const int *s_pos, int j0,
                      float c, int g, int r) {
        X8 pf[NK], df[NK];
        f32x4 pr[2][NK], ds[2][NK];
        float top[NK];
#pragma unroll
        for (int y = 0; y < NK; ++y) top[y] = 0.f;
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int y = 0; y < NK; ++y) pr[w][y] = ds[w][y] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < NS; ++x) {
            X8 v[NK];
#pragma unroll
            for (int y = 0; y < NK; ++y)
                if constexpr (VL)
                    v[y] = *(const X8 *)(sv + (y * 16 + r) * DP + swz<NC>(y * 16 + r, x * 4 + g) * 8);
                else
                    v[y] = vf[y][x];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const int j = j0 + w * 16 + r;
                const X8 qf = *(const X8 *)(sq + j * DP + swz<NC>(j, x * 4 + g) * 8);
                const X8 of = *(const X8 *)(so + j * DP + swz<NC>(j, x * 4 + g) * 8);
#pragma unroll
                for (int y = 0; y < NK; ++y) {
                    pr[w][y] = mfma(qf, kf[y][x], pr[w][y]);
                    ds[w][y] = mfma(of, v[y], ds[w][y]);
                }
            }
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const f32x4 lse = *(const f32x4 *)(s_lse + j0 + w * 16 + g * 4);
            const f32x4 delta = *(const f32x4 *)(s_delta + j0 + w * 16 + g * 4);
            const i32x4 pos = *(const i32x4 *)(s_pos + j0 + w * 16 + g * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int y = 0; y < NK; ++y) {
                    // three operations an element: cheaper than a second form
                    // of the loop for tiles without hidden pairs, whose copies
                    // of the sums do not fit the registers
                    const bool in = (uint32_t)(pos[i] - key[y]) <= span[y];
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(pr[w][y][i], c, -lse[i]));
                    const float p = in ? e : 0.f;
                    const float d = p * (ds[w][y][i] - delta[i]);
                    pf[y][w * 4 + i] = (T)p;
                    if constexpr (Range<T>::on) {
                        ds[w][y][i] = d;
                        top[y] = fmaxf(top[y], __builtin_fabsf(d));
                    } else {
                        df[y][w * 4 + i] = (T)d;
                    }
                }
        }
        if constexpr (Range<T>::on) {
            bool grow = false;
#pragma unroll
            for (int y = 0; y < NK; ++y) grow = grow | (top[y] > limit[y]);
            if (__any(grow)) {
#pragma unroll
                for (int y = 0; y < NK; ++y) {
                    const float most = max_rows(top[y]);
                    if (most > limit[y]) {
                        const float m = Range<T>::scale_for(most), f = mul[y] == 0.f ? 0.f : m / mul[y];
                        mul[y] = m, limit[y] = Range<T>::kTop / m;
#pragma unroll
                        for (int d = 0; d < ND; ++d) dk[d][y] *= f;
                    }
                }
            }
#pragma unroll
            for (int y = 0; y < NK; ++y)
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int i = 0; i < 4; ++i) df[y][w * 4 + i] = (T)(ds[w][y][i] * mul[y]);
        }
        // the wave that has its products ready goes first: its SIMD's other wave
        // is then in its exponentials (417 -> 407 us; at the scores' products
        // instead 452)
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const X8 of = columns<T, DP>(so, j0, d, g, r), qf = columns<T, DP>(sq, j0, d, g, r);
#pragma unroll
            for (int y = 0; y < NK; ++y) {
                dv[d][y] = mfma(of, pf[y], dv[d][y]);
                dk[d][y] = mfma(qf, df[y], dk[d][y]);
            }
        }
        __builtin_amdgcn_s_setprio(0);
    }
    // the sums in their own units
    LSMX_DEV float k_unit(int y) const {
        const float p = Range<T>::on ? 1.f / 1024.f : 1.f;
        return !Range<T>::on ? 1.f : mul[y] == 0.f ? 0.f : p / mul[y];
    }
    LSMX_DEV static float v_unit() { return Range<T>::on ? 1.f / 1024.f : 1.f; }
};

// Elements of one share's dK (or dV).
LSMX_DEV int64_t share_size(const AttnArgs &a) {
    return (a.offsets ? (int64_t)a.tokens : (int64_t)a.batch * a.k_len) * a.kv_heads * a.dim;
}

// The first token past the window of the key tile that holds key j.
LSMX_DEV int far_token(const AttnArgs &a, const Seq &s, int j, int keys) {
    return min(j / kKM * kKM + kKM, keys) - 1 + a.window - s.shift;
}

// Bound by the loads of the chunks' rows, each used for 16 keys only: 25 us at 2 x
// 4096 tokens, 32/8 heads of 128, window 1024, 4 sinks.
//
// Far rows: one chunk of rows, 16 sinks; the 4 waves take 32 rows each of a
// tile of 128 and are joined in LDS.  part: [16 sinks][key head][chunk][dK, dV][16][DP].
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_far_kernel(AttnArgs a) {
    constexpr int ND = DP / 16, NS = DP / 32;
    typedef typename Vec<T>::x8 X8;
    __shared__ __attribute__((aligned(16))) uint8_t smem[2 * kFar * DP * 2];
    __shared__ __attribute__((aligned(16))) float s_lse[kFar], s_delta[kFar];
    __shared__ __attribute__((aligned(16))) int s_pos[kFar];
    T *sq = (T *)smem, *so = sq + kFar * DP;

    const int slots = a.tiles, slot = uniform(blockIdx.x % slots), rest = uniform(blockIdx.x / slots);
    const int hkv = rest % a.kv_heads, group = rest / a.kv_heads;
    Seq s;
    if (!find_tile(a, slot, a.chunk, a.group, a.q_len, s)) return;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, r = lane & 15;
    const int keys = a.offsets ? s.q_len : s.k_len, rows = s.q_len * a.group, key = group * 16 + r;
    if (group * 16 >= keys) return;
    const int first = max(far_token(a, s, group * 16, keys), 0);
    if (first >= s.q_len) return;
    const int row_lo = max(s.tile * a.chunk, first * a.group), row_hi = min((s.tile + 1) * a.chunk, rows);
    if (row_lo >= row_hi) return;

    KeySums<T, DP, 1, false> sums;
    sums.init(a, key);
    const T *kp = (const T *)a.k + s.b * a.k_b + (s.k0 + key) * a.k_t + hkv * a.k_h;
    const T *vp = (const T *)a.v + s.b * a.v_b + (s.k0 + key) * a.v_t + hkv * a.v_h;
#pragma unroll
    for (int x = 0; x < NS; ++x) {
        const int c = x * 4 + g;
        const bool ok = key < keys && c * 8 < a.dim;
        sums.kf[0][x] = ok ? *(const X8 *)(kp + c * 8) : X8{};
        sums.vf[0][x] = ok ? *(const X8 *)(vp + c * 8) : X8{};
    }
    Rows<T, DP> in{a, s, hkv, row_hi};
    for (int row0 = row_lo; row0 < row_hi; row0 += kFar) {
        __syncthreads();
        in.fetch(row0, sq, so, kFar);
        if (threadIdx.x < kFar) in.stats(row0 + threadIdx.x, s_lse[threadIdx.x], s_delta[threadIdx.x], s_pos[threadIdx.x]);
        wait_dma();
        __syncthreads();
        // rows past their window see none but the sinks
        sums.add(sq, so, s_lse, s_delta, s_pos, wave * 32, a.c, g, r);
    }
    // join the waves: dK, then dV
    float *w_out = (float *)smem;  // [4][16][DP]
    float *part = a.part + ((int64_t)(group * a.kv_heads + hkv) * slots + slot) * 2 * 16 * DP;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const float f = v ? sums.v_unit() : sums.k_unit(0);
        __syncthreads();
#pragma unroll
        for (int d = 0; d < ND; ++d)
            *(f32x4 *)(w_out + (wave * 16 + r) * DP + d * 16 + g * 4) = (v ? sums.dv[d][0] : sums.dk[d][0]) * f;
        __syncthreads();
        for (int i = threadIdx.x * 4; i < 16 * DP; i += 1024) {
            f32x4 x = *(f32x4 *)(w_out + i);
#pragma unroll
            for (int w = 1; w < 4; ++w) x += *(f32x4 *)(w_out + w * 16 * DP + i);
            *(f32x4 *)(part + v * 16 * DP + i) = x;
        }
    }
}

// Rows (token, head) that see some key of tile `tile`, but for the far rows of
// sinks: [first, second).
struct RowSpan {
    int lo, hi;
};
LSMX_DEV RowSpan rows_of_keys(const AttnArgs &a, const Seq &s, int keys) {
    const int key0 = s.tile * kKM, key1 = min(key0 + kKM, keys) - 1;
    int hi = s.q_len;
    if (a.window && (a.chunk || key0 >= a.sinks)) hi = min(hi, key1 + a.window - s.shift);
    return RowSpan{max(0, key0 - s.shift) * a.group, max(hi, 0) * a.group};
}

// Each workgroup owns 128 keys, a wave 32 of them: K in registers, the sums of
// dK and dV in 128 more, the rows through LDS.  Few key tiles take their rows in
// shares, whose sums go to memory in fp32 and are joined by a kernel of its own.
//
// Bound by the two waves per SIMD that these registers leave: the vector unit is
// busy 54% of the time, the matrix unit 33%, LDS 36%, and what one wave waits for
// the other cannot always fill; 12% more is the sequence's end, whose keys fewer
// rows see.  2 x 4096 tokens, 32/8 heads of 128, window 1024: 407 us for four
// products = 593 TFLOP/s of the visible pairs.
//
// Head 128: two waves per SIMD only with V in LDS, tiles of 32 rows and the LDS
// places made anew each time (245 registers; with V in registers 320, one wave
// per SIMD: 484 us).
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void attn_dkv_kernel(AttnArgs a) {
    constexpr int NS = DP / 32, ND = DP / 16;
    constexpr bool VL = DP == 128;          // V in LDS
    constexpr int kKN = VL ? 32 : 64;       // rows of a tile
    typedef typename Vec<T>::x8 X8;
    typedef typename Vec<T>::x4 X4;
    __shared__ __attribute__((aligned(16))) T sq[2][kKN * DP], so[2][kKN * DP], s_v[VL ? kKM * DP : 8];
    __shared__ __attribute__((aligned(16))) float s_lse[2][kKN], s_delta[2][kKN];
    __shared__ __attribute__((aligned(16))) int s_pos[2][kKN];

    const Item item = item_of(a, a.shares);
    const int hkv = item.head, share = item.share;
    if (hkv >= a.kv_heads) return;
    Seq s;
    if (!find_tile(a, item.tile, kKM, 1, a.k_len, s)) return;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, r = lane & 15;
    const int keys = a.offsets ? s.q_len : s.k_len;  // of a dead sequence too
    const int key0 = s.tile * kKM, key1 = min(key0 + kKM, keys) - 1;

    const RowSpan all = rows_of_keys(a, s, keys);
    int row_lo = all.lo, row_hi = all.hi;
    if (a.shares > 1) {
        if (share && (int64_t)share * a.share_rows >= row_hi - row_lo) return;
        row_lo += share * a.share_rows;
        row_hi = min(row_hi, row_lo + a.share_rows);
    }
    Rows<T, DP> in{a, s, hkv, row_hi};
    if (row_lo < row_hi) {
        in.fetch(row_lo, sq[0], so[0], kKN);
        if (threadIdx.x < kKN) in.stats(row_lo + threadIdx.x, s_lse[0][threadIdx.x], s_delta[0][threadIdx.x], s_pos[0][threadIdx.x]);
    }

    KeySums<T, DP, 2, VL> sums;
    sums.init(a, key0 + wave * 32 + r);
    const int(&key)[2] = sums.key;
    if constexpr (VL) {
        const T *vp = (const T *)a.v + s.b * a.v_b + (s.k0 + key0) * a.v_t + hkv * a.v_h;
        const int left = keys - key0, dim = a.dim, v_t = (int)a.v_t;
        fetch_rows<T, DP>(buf_rsrc(vp, 0x7FFFFFFF), s_v, kKM, [=](int j, int c) {
            return j < left && c * 8 < dim ? (uint32_t)(j * v_t + c * 8) * 2 : kZeros;
        });
        sums.sv = s_v + wave * 32 * DP;
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        const T *kp = (const T *)a.k + s.b * a.k_b + (s.k0 + key[y]) * a.k_t + hkv * a.k_h;
        const T *vp = (const T *)a.v + s.b * a.v_b + (s.k0 + key[y]) * a.v_t + hkv * a.v_h;
#pragma unroll
        for (int x = 0; x < NS; ++x) {
            const int c = x * 4 + g;
            const bool ok = key[y] < keys && c * 8 < a.dim;
            sums.kf[y][x] = ok ? *(const X8 *)(kp + c * 8) : X8{};
            if constexpr (!VL) sums.vf[y][x] = ok ? *(const X8 *)(vp + c * 8) : X8{};
        }
    }
    const int wkey0 = key0 + wave * 32, wkey1 = wkey0 + 31;
    wait_dma();
    __syncthreads();
    int n = 0;
    for (int row0 = row_lo; row0 < row_hi; row0 += kKN, n ^= 1) {
        const bool more = row0 + kKN < row_hi;
        float lse = 0.f, delta = 0.f;
        int pos = -1;
        if (more) {
            if (threadIdx.x < kKN) in.stats(row0 + kKN + threadIdx.x, lse, delta, pos);
            in.fetch(row0 + kKN, sq[n ^ 1], so[n ^ 1], kKN);
        }
        // hidden from every row
        const int pmin = div_by(row0, a.by_group) + s.shift, pmax = div_by(min(row0 + kKN, row_hi) - 1, a.by_group) + s.shift;
        const bool none = wkey0 > pmax || wkey0 > key1 || (a.window && wkey1 <= pmin - a.window && wkey0 >= a.sinks);
        if (!none) {
#pragma unroll
            for (int u = 0; u < kKN / 32; ++u) {
                int lr = r;
                if constexpr (VL) asm volatile("" : "+v"(lr));
                sums.add(sq[n], so[n], s_lse[n], s_delta[n], s_pos[n], u * 32, a.c, g, lr);
            }
        }
        wait_dma();
        if (more && threadIdx.x < kKN) s_lse[n ^ 1][threadIdx.x] = lse, s_delta[n ^ 1][threadIdx.x] = delta, s_pos[n ^ 1][threadIdx.x] = pos;
        __syncthreads();
    }

#pragma unroll
    for (int y = 0; y < 2; ++y) {
        const float fk = sums.k_unit(y), fv = sums.v_unit();
#pragma unroll
        for (int d = 0; d < ND; ++d) sums.dk[d][y] *= fk, sums.dv[d][y] *= fv;
        const int group = (wkey0 + y * 16) / 16;
        if (a.chunk && share == 0 && wkey0 + y * 16 < min(a.sinks, keys)) {
            const int first = max(far_token(a, s, wkey0, keys), 0) * a.group, rows = s.q_len * a.group;
            const int slot0 = first_tile(a, s, a.chunk, a.group);
            for (int c = first / a.chunk; c * a.chunk < rows && first < rows; ++c) {
                const float *part = a.part + ((int64_t)(group * a.kv_heads + hkv) * a.far_slots + slot0 + c) * 2 * 16 * DP + r * DP + g * 4;
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    sums.dk[d][y] += *(const f32x4 *)(part + d * 16);
                    sums.dv[d][y] += *(const f32x4 *)(part + 16 * DP + d * 16);
                }
            }
        }
        if (key[y] >= keys) continue;
        const int64_t at = (((a.offsets ? s.k0 : (int64_t)s.b * a.k_len) + key[y]) * a.kv_heads + hkv) * a.dim;
        if (a.shares > 1) {
            const int64_t one = share_size(a);
            float *to = a.share_part + 2 * share * one + at;
#pragma unroll
            for (int d = 0; d < ND; ++d)
                if (d * 16 + g * 4 < a.dim) {
                    *(f32x4 *)(to + d * 16 + g * 4) = sums.dk[d][y];
                    *(f32x4 *)(to + one + d * 16 + g * 4) = sums.dv[d][y];
                }
            continue;
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            X4 wk, wv;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                wk[i] = (T)(sums.dk[d][y][i] * a.scale);
                wv[i] = (T)sums.dv[d][y][i];
            }
            if (d * 16 + g * 4 < a.dim) {
                *(X4 *)((T *)a.dk + at + d * 16 + g * 4) = wk;
                *(X4 *)((T *)a.dv + at + d * 16 + g * 4) = wv;
            }
        }
    }
}

// Joins the shares of 16 keys, in their order.  Bound by the shares' bytes: 13
// of 5086 keys of 4 heads of 128, half of them empty, 26 us = 5 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    typedef typename Vec<T>::x4 X4;
    const int item = blockIdx.x / 8, hkv = item / a.tiles;
    Seq s;
    if (!find_tile(a, item - hkv * a.tiles, kKM, 1, a.k_len, s)) return;
    const int keys = a.offsets ? s.q_len : s.k_len, key0 = s.tile * kKM + (blockIdx.x & 7) * 16;
    const RowSpan all = rows_of_keys(a, s, keys);
    const int n = max(1, (all.hi - all.lo + a.share_rows - 1) / a.share_rows), quads = a.dim / 4;
    const int64_t one = share_size(a);
    for (int i = threadIdx.x; i < 16 * quads; i += 256) {
        const int j = i / quads, key = key0 + j;
        if (key >= keys) return;
        const int64_t at = (((a.offsets ? s.k0 : (int64_t)s.b * a.k_len) + key) * a.kv_heads + hkv) * a.dim + (i - j * quads) * 4;
        f32x4 dk{0, 0, 0, 0}, dv{0, 0, 0, 0};
#pragma unroll 4
        for (int c = 0; c < n; ++c) {
            const float *p = a.share_part + 2 * c * one + at;
            dk += *(const f32x4 *)p;
            dv += *(const f32x4 *)(p + one);
        }
        X4 wk, wv;
#pragma unroll
        for (int e = 0; e < 4; ++e) wk[e] = (T)(dk[e] * a.scale), wv[e] = (T)dv[e];
        *(X4 *)((T *)a.dk + at) = wk;
        *(X4 *)((T *)a.dv + at) = wv;
    }
}

// The far rows' chunks: enough of them to spread a sequence over 64 workgroups,
// none below 512 rows.  Past 256 sinks their tiles are no exception any more,
// and take all rows themselves.
struct Far {
    int chunk, slots, groups;
    int64_t bytes;
};
Far far_plan(const AttnArgs &a) {
    Far f{};
    if (!a.window || !a.sinks || a.sinks > 256) return f;
    const int64_t rows = (int64_t)(a.offsets ? a.tokens : a.q_len) * a.group;
    if (rows <= (int64_t)a.window * a.group) return f;
    f.chunk = (int)((rows / 64 + 127) / 128 * 128);
    if (f.chunk < 512) f.chunk = 512;
    f.slots = (int)((rows + f.chunk - 1) / f.chunk);
    f.slots = a.offsets ? f.slots + a.batch + 2 : f.slots * a.batch;
    f.groups = (a.sinks + 15) / 16;
    f.bytes = (int64_t)f.groups * a.kv_heads * f.slots * 2 * 16 * (a.dim <= 64 ? 64 : 128) * 4;
    return f;
}
// Shares of the rows of key tiles: where the longest tile would take over half as
// long again as the chip for all, about 1024 workgroups in equal parts, none
// below 512 rows, and the sums of no more than 512 MiB.  Causal, without and with:
// 5506 tokens of 5/1 heads of 64, 924 us and 106 + 13 to join; 5086 of 32/4 of 128,
// 2444 and 750 + 26; 517 of 8/2 of 128, 129 and 39 + 4.  A window's equal tiles gain
// 12% at most and are left alone where they fill the chip.
struct Shares {
    int n, rows;
    int64_t bytes;
};
Shares share_plan(const AttnArgs &a, const Far &far) {
    Shares p{1, 0, 0};
    const int64_t keys = a.offsets ? a.tokens : (int64_t)a.batch * a.k_len, seqs = a.batch > 0 ? a.batch : 1;
    const int64_t own = a.offsets ? a.tokens / seqs : a.q_len, most = a.offsets ? a.tokens : a.q_len;
    const bool windowed = a.window && (far.chunk || !a.sinks);
    // rows of the longest tile, and of all: a tile's reach, or half the sequence
    const int64_t reach = (int64_t)a.window + kKM, longest = (windowed && reach < most ? reach : most) * a.group;
    const int64_t mean = (windowed && reach < own / 2 ? reach : (own + 1) / 2) * a.group;
    const int64_t total = (keys + kKM - 1) / kKM * a.kv_heads * mean;
    if (!keys || !total || longest <= 512 || longest * 512 < total + total / 2) return p;
    const int64_t one = keys * a.kv_heads * a.dim * 8, room = (int64_t)512 << 20;
    int64_t rows = (total / 1024 + 127) / 128 * 128;
    if (rows < 512) rows = 512;
    if ((longest + rows - 1) / rows * one > room) {
        const int64_t n = room / one;
        if (n < 2) return p;
        rows = ((longest + n - 1) / n + 127) / 128 * 128;
    }
    const int64_t n = (longest + rows - 1) / rows;
    if ((keys / kKM + a.batch + 2) * a.kv_heads * n >= (int64_t)1 << 27) return p;
    p.n = (int)n;
    p.rows = (int)rows;
    p.bytes = p.n > 1 ? p.n * one : 0;
    return p;
}
int64_t delta_bytes(const AttnArgs &a) {
    const int64_t rows = (a.offsets ? (int64_t)a.tokens : (int64_t)a.batch * a.q_len) * a.heads;
    return (4 * rows + 255) / 256 * 256;
}

template <typename T, int DP>
hipError_t bwd(const AttnArgs &in, hipStream_t s) {
    AttnArgs a = in;
    const Far far = far_plan(a);
    a.part = (float *)((uint8_t *)a.delta + delta_bytes(a));
    const int pad = a.offsets ? a.batch + 2 : 0, many = a.offsets ? 1 : a.batch;
    const int tokens = a.offsets ? a.tokens : a.q_len;
    if (tokens) {
        const int64_t rows = (int64_t)tokens * a.group;
        // 32 rows a wave where that gives each CU a workgroup, else 16, which read
        // twice as much of LDS per product: 216 and 252 workgroups of 128 rows (5506
        // tokens of 5/1 heads of 64; 3 x 777 of 12, window 256, fp16) took 138 and 26
        // us, 111 and 21 as twice as many of 64; 264 took 82 both, 536 took 39, 41
        const bool wide = (rows + 127) / 128 * many * a.kv_heads >= 256;
        a.tiles = (int)(wide ? (rows + 127) / 128 : (rows + 63) / 64) * many + pad;
        if (wide)
            attn_dq_kernel<T, DP, 2><<<order_items(a, (int64_t)a.tiles * a.kv_heads), 256, 0, s>>>(a);
        else
            attn_dq_kernel<T, DP, 1><<<order_items(a, (int64_t)a.tiles * a.kv_heads), 256, 0, s>>>(a);
        if (far.chunk) {
            a.chunk = far.chunk, a.tiles = a.far_slots = far.slots;
            attn_far_kernel<T, DP><<<(unsigned)far.slots * a.kv_heads * far.groups, 256, 0, s>>>(a);
        }
    }
    a.tiles = ((a.offsets ? a.tokens : a.k_len) + kKM - 1) / kKM * many + pad;
    if (!a.tiles) return hipGetLastError();
    const Shares shares = share_plan(a, far);
    a.shares = shares.n, a.share_rows = shares.rows;
    a.share_part = (float *)((uint8_t *)a.part + far.bytes);
    attn_dkv_kernel<T, DP><<<order_items(a, (int64_t)a.tiles * a.kv_heads * a.shares), 256, 0, s>>>(a);
    if (a.shares > 1) attn_join_kernel<T><<<(unsigned)(a.tiles * a.kv_heads * 8), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

int64_t attn_bwd_workspace(const AttnArgs &a) {
    const Far far = far_plan(a);
    return delta_bytes(a) + far.bytes + share_plan(a, far).bytes + 256;
}

hipError_t launch_attn_bwd(const AttnArgs &a, int dtype, hipStream_t s) {
    if (dtype == LSMX_BF16) return a.dim <= 64 ? bwd<__bf16, 64>(a, s) : bwd<__bf16, 128>(a, s);
    return a.dim <= 64 ? bwd<_Float16, 64>(a, s) : bwd<_Float16, 128>(a, s);
}

}  // namespace lsmx
