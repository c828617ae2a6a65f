// Attention with a sliding window and sinks: gradients.
//
//   P_ij = exp(s_ij - lse_i),  dV_j = sum_i P_ij dO_i,
//   dS_ij = P_ij (dO_i . v_j - delta_i),  delta_i = dO_i . o_i,
//   dQ_i = scale sum_j dS_ij k_j,  dK_j = scale sum_i dS_ij q_i.
//
// Two kernels, so that every sum has one owner and one order (no atomics): one
// owns rows and runs over their keys (dQ), the other owns keys and runs over
// the rows of all heads that share them (dK, dV).  Both recompute S and dP:
// seven products where one kernel with shared accumulators would take five.
#include "lsmx_attn.h"

namespace lsmx {
namespace {

constexpr int kBM = 128;  // dQ: rows of a workgroup
constexpr int kBN = 64;   // dQ: keys of a tile
constexpr int kKM = 128;  // dK, dV: keys of a workgroup
constexpr int kKN = 64;   // dK, dV: rows of a tile

// delta of every row: 16 lanes per row.
template <typename T>
__global__ __launch_bounds__(256) void attn_delta_kernel(AttnArgs a) {
    typedef typename Vec<T>::x8 X8;
    const int64_t tokens = a.offsets ? a.tokens : (int64_t)a.batch * a.q_len;
    const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int r = threadIdx.x & 15;
    if (row >= tokens * a.heads) return;
    const int64_t tok = row / a.heads;
    const int h = (int)(row - tok * a.heads);
    const int b = a.offsets ? 0 : (int)(tok / a.q_len);
    const int64_t t = a.offsets ? tok : tok - (int64_t)b * a.q_len;
    float sum = 0.f;
    if (r * 8 < a.dim) {
        const X8 x = *(const X8 *)((const T *)a.d_o + b * a.do_b + t * a.do_t + h * a.do_h + r * 8);
        const X8 y = *(const X8 *)((const T *)a.o + b * a.o_b + t * a.o_t + h * a.o_h + r * 8);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = __builtin_fmaf((float)x[i], (float)y[i], sum);
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor(sum, d);
    if (r == 0) a.delta[b * a.lse_b + h * a.lse_h + t] = sum;
}

// Stages 64 rows of two tensors (strides per key row, or per token and head).
template <typename T, int DP>
struct Stage {
    static constexpr int NC = DP / 8, NU = 64 * NC / 256;
    u32x4 x[NU], y[NU];
    LSMX_DEV void store(T *sx, T *sy) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int id = threadIdx.x + 256 * u, j = id / NC, c = id % NC;
            *(u32x4 *)(sx + j * DP + swz<NC>(j, c) * 8) = x[u];
            *(u32x4 *)(sy + j * DP + swz<NC>(j, c) * 8) = y[u];
        }
    }
};

template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_dq_kernel(AttnArgs a) {
    constexpr int NC = DP / 8, NS = DP / 32, ND = DP / 16;
    typedef typename Vec<T>::x8 X8;
    typedef typename Vec<T>::x4 X4;
    __shared__ T sk[kBN * DP], sv[kBN * DP];

    const int item = xcd_item(blockIdx.x, a.per);
    if (item >= a.tiles * a.kv_heads) return;
    const int hkv = item / a.tiles;
    Seq s;
    if (!find_tile(a, a.tiles - 1 - item % a.tiles, kBM, a.group, a.q_len, s)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int row0 = s.tile * kBM, rows = s.q_len * a.group;

    int pos[2];
    int64_t q_at[2];
    float lse[2], delta[2];
    X8 qf[2][NS], of[2][NS];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int row = row0 + wave * 32 + r + 16 * t;
        const bool in = row < rows;
        const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
        pos[t] = in ? tok + s.shift : -1;
        const int64_t l_at = s.b * a.lse_b + h * a.lse_h + s.q0 + tok;
        lse[t] = in ? a.lse[l_at] : 0.f;
        delta[t] = in ? a.delta[l_at] : 0.f;
        const int64_t token = (a.offsets ? s.q0 : (int64_t)s.b * a.q_len) + tok;
        q_at[t] = in ? (token * a.heads + h) * a.dim : -1;
        const T *qp = (const T *)a.q + s.b * a.q_b + (s.q0 + tok) * a.q_t + h * a.q_h;
        const T *op = (const T *)a.d_o + s.b * a.do_b + (s.q0 + tok) * a.do_t + h * a.do_h;
#pragma unroll
        for (int x = 0; x < NS; ++x) {
            const int c = x * 4 + g;
            const bool ok = in && c * 8 < a.dim;
            qf[t][x] = ok ? *(const X8 *)(qp + c * 8) : X8{};
            of[t][x] = ok ? *(const X8 *)(op + c * 8) : X8{};
        }
    }
    f32x4 dq[ND][2];
#pragma unroll
    for (int d = 0; d < ND; ++d) dq[d][0] = dq[d][1] = f32x4{0, 0, 0, 0};

    const int pmin = div_by(row0, a.by_group) + s.shift;
    const int pmax = div_by(min(row0 + kBM, rows) - 1, a.by_group) + s.shift;
    const int hi = min(pmax + 1, s.k_len), lo = a.window ? max(0, pmin - a.window + 1) : 0;
    const int t_sink = (min(a.sinks, hi) + kBN - 1) / kBN, t_hi = hi > 0 ? (hi + kBN - 1) / kBN : 0;
    const int t_lo = lo / kBN;
    auto next = [&](int t) { return t + 1 < t_sink ? t + 1 : max(t + 1, t_lo); };
    int t = t_sink > 0 ? 0 : t_lo;

    const T *kp = (const T *)a.k + s.b * a.k_b + s.k0 * a.k_t + hkv * a.k_h;
    const T *vp = (const T *)a.v + s.b * a.v_b + s.k0 * a.v_t + hkv * a.v_h;
    Stage<T, DP> kv;
    auto load = [&](int j0) {
#pragma unroll
        for (int u = 0; u < Stage<T, DP>::NU; ++u) {
            const int id = threadIdx.x + 256 * u, j = j0 + id / NC, c = id % NC;
            const bool in = j < s.k_len && c * 8 < a.dim;
            kv.x[u] = in ? *(const u32x4 *)(kp + j * a.k_t + c * 8) : u32x4{0, 0, 0, 0};
            kv.y[u] = in ? *(const u32x4 *)(vp + j * a.v_t + c * 8) : u32x4{0, 0, 0, 0};
        }
    };
    if (t < t_hi) load(t * kBN);
    while (t < t_hi) {
        const int j0 = t * kBN, tn = next(t);
        __syncthreads();
        kv.store(sk, sv);
        __syncthreads();
        if (tn < t_hi) load(tn * kBN);
        const bool full = j0 + kBN - 1 <= pmin && (!a.window || j0 > pmax - a.window || j0 + kBN - 1 < a.sinks);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            X8 df[2];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const int kt = u * 2 + w, j = kt * 16 + r;
                f32x4 st[2], dp[2];
                st[0] = st[1] = dp[0] = dp[1] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int x = 0; x < NS; ++x) {
                    const X8 kf = *(const X8 *)(sk + j * DP + swz<NC>(j, x * 4 + g) * 8);
                    const X8 vf = *(const X8 *)(sv + j * DP + swz<NC>(j, x * 4 + g) * 8);
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        st[y] = mfma(kf, qf[y][x], st[y]);
                        dp[y] = mfma(vf, of[y][x], dp[y]);
                    }
                }
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int jj = j0 + kt * 16 + g * 4 + i;
                        const float ds = __builtin_amdgcn_exp2f(__builtin_fmaf(st[y][i], a.c, -lse[y])) * (dp[y][i] - delta[y]);
                        const bool in = full | sees(jj, pos[y], window_low(pos[y], a.window), a.sinks);
                        df[y][w * 4 + i] = (T)(in ? ds : 0.f);
                    }
            }
            const int j = u * 32 + g * 4 + (r >> 2);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const int c = d * 2 + ((r & 3) >> 1), e = (r & 1) * 4;
                const X8 kf = join<X4, X8>(read_tr<T>(sk + j * DP + swz<NC>(j, c) * 8 + e),
                                           read_tr<T>(sk + (j + 16) * DP + swz<NC>(j + 16, c) * 8 + e));
                dq[d][0] = mfma(kf, df[0], dq[d][0]);
                dq[d][1] = mfma(kf, df[1], dq[d][1]);
            }
        }
        t = tn;
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        if (q_at[y] < 0) continue;
        T *p = (T *)a.dq + q_at[y];
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            X4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (T)(dq[d][y][i] * a.scale);
            if (d * 16 + g * 4 < a.dim) *(X4 *)(p + d * 16 + g * 4) = w;
        }
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_dkv_kernel(AttnArgs a) {
    constexpr int NC = DP / 8, NS = DP / 32, ND = DP / 16;
    typedef typename Vec<T>::x8 X8;
    typedef typename Vec<T>::x4 X4;
    __shared__ T sq[kKN * DP], so[kKN * DP];
    __shared__ float s_lse[kKN], s_delta[kKN];
    __shared__ int s_pos[kKN];

    const int item = xcd_item(blockIdx.x, a.per);
    if (item >= a.tiles * a.kv_heads) return;
    const int hkv = item / a.tiles;
    Seq s;
    if (!find_tile(a, item % a.tiles, kKM, 1, a.k_len, s)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int keys = a.offsets ? s.q_len : s.k_len;  // of a dead sequence too
    const int key0 = s.tile * kKM;

    X8 kf[2][NS], vf[2][NS];
    int key[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        key[t] = key0 + wave * 32 + t * 16 + r;
        const T *kp = (const T *)a.k + s.b * a.k_b + (s.k0 + key[t]) * a.k_t + hkv * a.k_h;
        const T *vp = (const T *)a.v + s.b * a.v_b + (s.k0 + key[t]) * a.v_t + hkv * a.v_h;
#pragma unroll
        for (int x = 0; x < NS; ++x) {
            const int c = x * 4 + g;
            const bool ok = key[t] < keys && c * 8 < a.dim;
            kf[t][x] = ok ? *(const X8 *)(kp + c * 8) : X8{};
            vf[t][x] = ok ? *(const X8 *)(vp + c * 8) : X8{};
        }
    }
    f32x4 dk[ND][2], dv[ND][2];
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d][0] = dk[d][1] = dv[d][0] = dv[d][1] = f32x4{0, 0, 0, 0};

    // the rows that see some key of the tile
    const int key1 = min(key0 + kKM, keys) - 1;
    const int tok_lo = max(0, key0 - s.shift);
    int tok_hi = s.q_len;
    if (a.window && key0 >= a.sinks) tok_hi = min(tok_hi, key1 + a.window - s.shift);
    const int row_lo = tok_lo * a.group, row_hi = max(tok_hi, 0) * a.group;

    Stage<T, DP> qo;
    float lse_r = 0.f, delta_r = 0.f;
    int pos_r = -1;
    auto load = [&](int row0) {
#pragma unroll
        for (int u = 0; u < Stage<T, DP>::NU; ++u) {
            const int id = threadIdx.x + 256 * u, row = row0 + id / NC, c = id % NC;
            const bool in = row < row_hi;
            const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
            const bool ok = in && c * 8 < a.dim;
            qo.x[u] = ok ? *(const u32x4 *)((const T *)a.q + s.b * a.q_b + (s.q0 + tok) * a.q_t + h * a.q_h + c * 8)
                         : u32x4{0, 0, 0, 0};
            qo.y[u] = ok ? *(const u32x4 *)((const T *)a.d_o + s.b * a.do_b + (s.q0 + tok) * a.do_t + h * a.do_h + c * 8)
                         : u32x4{0, 0, 0, 0};
        }
        if (threadIdx.x < kKN) {
            const int row = row0 + threadIdx.x;
            const bool in = row < row_hi;
            const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
            const int64_t l_at = s.b * a.lse_b + h * a.lse_h + s.q0 + tok;
            lse_r = in ? a.lse[l_at] : 0.f;
            delta_r = in ? a.delta[l_at] : 0.f;
            pos_r = in ? tok + s.shift : -1;
        }
    };
    if (row_lo < row_hi) load(row_lo);
    for (int row0 = row_lo; row0 < row_hi; row0 += kKN) {
        __syncthreads();
        qo.store(sq, so);
        if (threadIdx.x < kKN) s_lse[threadIdx.x] = lse_r, s_delta[threadIdx.x] = delta_r, s_pos[threadIdx.x] = pos_r;
        __syncthreads();
        if (row0 + kKN < row_hi) load(row0 + kKN);
        const int pmin = div_by(row0, a.by_group) + s.shift;
        const int pmax = div_by(min(row0 + kKN, row_hi) - 1, a.by_group) + s.shift;
        const bool full = row0 + kKN <= row_hi && key1 == key0 + kKM - 1 && key1 <= pmin &&
                          (!a.window || key0 > pmax - a.window || key1 < a.sinks);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            X8 pf[2], df[2];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const int rt = u * 2 + w, j = rt * 16 + r;
                f32x4 st[2], dp[2];
                st[0] = st[1] = dp[0] = dp[1] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int x = 0; x < NS; ++x) {
                    const X8 qf = *(const X8 *)(sq + j * DP + swz<NC>(j, x * 4 + g) * 8);
                    const X8 of = *(const X8 *)(so + j * DP + swz<NC>(j, x * 4 + g) * 8);
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        st[y] = mfma(qf, kf[y][x], st[y]);
                        dp[y] = mfma(of, vf[y][x], dp[y]);
                    }
                }
                const f32x4 lse = *(const f32x4 *)(s_lse + rt * 16 + g * 4);
                const f32x4 delta = *(const f32x4 *)(s_delta + rt * 16 + g * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int p = full ? 0 : s_pos[rt * 16 + g * 4 + i];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(st[y][i], a.c, -lse[i]));
                        const float ds = pr * (dp[y][i] - delta[i]);
                        const bool in = full | sees(key[y], p, window_low(p, a.window), a.sinks);
                        pf[y][w * 4 + i] = (T)(in ? pr : 0.f);
                        df[y][w * 4 + i] = (T)(in ? ds : 0.f);
                    }
                }
            }
            const int j = u * 32 + g * 4 + (r >> 2);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const int c = d * 2 + ((r & 3) >> 1), e = (r & 1) * 4;
                const X8 of = join<X4, X8>(read_tr<T>(so + j * DP + swz<NC>(j, c) * 8 + e),
                                           read_tr<T>(so + (j + 16) * DP + swz<NC>(j + 16, c) * 8 + e));
                const X8 qf = join<X4, X8>(read_tr<T>(sq + j * DP + swz<NC>(j, c) * 8 + e),
                                           read_tr<T>(sq + (j + 16) * DP + swz<NC>(j + 16, c) * 8 + e));
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    dv[d][y] = mfma(of, pf[y], dv[d][y]);
                    dk[d][y] = mfma(qf, df[y], dk[d][y]);
                }
            }
        }
    }
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        if (key[y] >= keys) continue;
        const int64_t at = (((a.offsets ? s.k0 : (int64_t)s.b * a.k_len) + key[y]) * a.kv_heads + hkv) * a.dim;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            X4 wk, wv;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                wk[i] = (T)(dk[d][y][i] * a.scale);
                wv[i] = (T)dv[d][y][i];
            }
            if (d * 16 + g * 4 < a.dim) {
                *(X4 *)((T *)a.dk + at + d * 16 + g * 4) = wk;
                *(X4 *)((T *)a.dv + at + d * 16 + g * 4) = wv;
            }
        }
    }
}

template <typename T, int DP>
hipError_t bwd(const AttnArgs &in, hipStream_t s) {
    AttnArgs a = in;
    const int64_t rows = (a.offsets ? (int64_t)a.tokens : (int64_t)a.batch * a.q_len) * a.heads;
    if (rows) attn_delta_kernel<T><<<(unsigned)((rows + 15) / 16), 256, 0, s>>>(a);
    const int pad = a.offsets ? a.batch + 2 : 0, many = a.offsets ? 1 : a.batch;
    a.tiles = (int)(((int64_t)(a.offsets ? a.tokens : a.q_len) * a.group + kBM - 1) / kBM) * many + pad;
    a.per = (int)(((int64_t)a.tiles * a.kv_heads + 7) / 8);
    if (rows) attn_dq_kernel<T, DP><<<(unsigned)a.per * 8, 256, 0, s>>>(a);
    a.tiles = ((a.offsets ? a.tokens : a.k_len) + kKM - 1) / kKM * many + pad;
    a.per = (int)(((int64_t)a.tiles * a.kv_heads + 7) / 8);
    if (a.tiles) attn_dkv_kernel<T, DP><<<(unsigned)a.per * 8, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

int64_t attn_bwd_workspace(const AttnArgs &a) {
    const int64_t rows = (a.offsets ? (int64_t)a.tokens : (int64_t)a.batch * a.q_len) * a.heads;
    return (4 * rows + 255) / 256 * 256 + 256;
}

hipError_t launch_attn_bwd(const AttnArgs &a, int dtype, hipStream_t s) {
    if (dtype == LSMX_BF16) return a.dim <= 64 ? bwd<__bf16, 64>(a, s) : bwd<__bf16, 128>(a, s);
    return a.dim <= 64 ? bwd<_Float16, 64>(a, s) : bwd<_Float16, 128>(a, s);
}

}  // namespace lsmx
