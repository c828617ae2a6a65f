// Attention with a sliding window and sinks: forward.
//
//   s_ij = scale q_i . k_j over the keys j that row i sees,
//   o_i  = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),
//
// in one pass over the keys with the running maximum m and sum of each row.
// The rows of a workgroup are (token, head) pairs that share a key head, token
// major, so grouped heads read their keys once.
//
// Layout (v_mfma_*_16x16x32, lane 16g + r):
//   S^T = K Q^T: keys are the rows of C, so a lane holds 4 keys (4g..4g+3) of
//   each 16 for one query row r; the softmax of a row lives in 4 lanes, and the
//   pair of key tiles 2u, 2u+1 gives the lane 8 probabilities that are, as they
//   stand, the B operand of O^T += V^T P^T when V^T's contraction runs over the
//   same 8 keys.  The transposing LDS read delivers exactly those.  No
//   probability crosses a lane, and O is rescaled lane by lane.
#include "lsmx_attn.h"

namespace lsmx {
namespace {

constexpr int kBM = 128;  // rows of a workgroup, 32 of each of 4 waves
constexpr int kBN = 64;   // keys of a tile

// Keys and values as they lie in memory, staged through registers into LDS.
template <typename T, int DP>
struct DenseKV {
    static constexpr int NC = DP / 8, NU = kBN * NC / 256;
    static constexpr bool kHoles = false;
    typedef AttnArgs Args;
    LSMX_DEV static const AttnArgs &attn(const Args &a) { return a; }
    LSMX_DEV static bool find(const Args &a, int t, Seq &s) {
        // the last tile of a sequence first: under a causal mask it is the longest
        return find_tile(a, a.tiles - 1 - t, kBM, a.group, a.q_len, s);
    }
    const T *k, *v;
    int64_t k_t, v_t;
    int k_len, dim;
    u32x4 kr[NU], vr[NU];

    LSMX_DEV void init(const AttnArgs &a, const Seq &s, int hkv) {
        k = (const T *)a.k + s.b * a.k_b + s.k0 * a.k_t + hkv * a.k_h;
        v = (const T *)a.v + s.b * a.v_b + s.k0 * a.v_t + hkv * a.v_h;
        k_t = a.k_t, v_t = a.v_t, k_len = s.k_len, dim = a.dim;
    }
    LSMX_DEV void load(int j0) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int id = threadIdx.x + 256 * u, j = j0 + id / NC, c = id % NC;
            const bool in = j < k_len && c * 8 < dim;
            kr[u] = in ? *(const u32x4 *)(k + j * k_t + c * 8) : u32x4{0, 0, 0, 0};
            vr[u] = in ? *(const u32x4 *)(v + j * v_t + c * 8) : u32x4{0, 0, 0, 0};
        }
    }
    LSMX_DEV void store(T *sk, T *sv) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int id = threadIdx.x + 256 * u, j = id / NC, c = id % NC;
            *(u32x4 *)(sk + j * DP + swz<NC>(j, c) * 8) = kr[u];
            *(u32x4 *)(sv + j * DP + swz<NC>(j, c) * 8) = vr[u];
        }
    }
};

// Keys and values of a paged MXFP4 cache, expanded to bf16 on their way into
// LDS (exact).  A thread takes a quarter of one key's and one value's vector.
template <int DP>
struct PagedKV {
    static constexpr int NC = DP / 8, NW = DP / 32;  // words of codes of a thread
    static constexpr bool kHoles = true;
    typedef AttendArgs Args;
    typedef __bf16 T;
    const Pool *p;
    int b, h, k_len, row, part;
    uint32_t kr[NW], vr[NW];
    uint32_t ke, ve;
    bool in;

    LSMX_DEV static const AttnArgs &attn(const Args &a) { return a.a; }
    LSMX_DEV static bool find(const Args &x, int t, Seq &s) {
        const AttnArgs &a = x.a;
        const int per = (a.q_len * a.group + kBM - 1) / kBM;
        t = a.tiles - 1 - t;
        s.b = t / per;
        s.tile = t - s.b * per;
        s.q_len = a.q_len;
        s.k_len = x.p.length(s.b);
        s.shift = s.k_len - s.q_len;
        s.q0 = s.k0 = 0;
        return true;
    }
    LSMX_DEV void init(const Args &a, const Seq &s, int hkv) {
        p = &a.p, b = s.b, h = hkv, k_len = s.k_len, row = threadIdx.x >> 2, part = threadIdx.x & 3;
    }
    LSMX_DEV void load(int j0) {
        const int j = j0 + row, pg = j < k_len ? p->page_of(b, j) : -1;
        in = pg >= 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) kr[i] = vr[i] = 0;
        ke = ve = 0;
        if (in) {
            const int64_t v = p->vec(pg, h, j);
            const uint8_t *kp = p->kc + v * (DP / 2) + part * (DP / 8), *vp = p->vc + v * (DP / 2) + part * (DP / 8);
            if constexpr (NW == 4) {
                *(u32x4 *)kr = *(const u32x4 *)kp;
                *(u32x4 *)vr = *(const u32x4 *)vp;
            } else {
                *(u32x2 *)kr = *(const u32x2 *)kp;
                *(u32x2 *)vr = *(const u32x2 *)vp;
            }
            const int blk = part * (DP / 32) / 4;
            ke = p->ks[v * (DP / 32) + blk];
            ve = p->vs[v * (DP / 32) + blk];
        }
    }
    LSMX_DEV void store(T *sk, T *sv) {
        const float ksc = e8m0_to_f32(ke), vsc = e8m0_to_f32(ve);
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int c = swz<NC>(row, part * NW + i);
            *(bf16x8 *)(sk + row * DP + c * 8) = fp4x8_to_bf16(kr[i], ksc);
            *(bf16x8 *)(sv + row * DP + c * 8) = fp4x8_to_bf16(vr[i], vsc);
        }
    }
};

// TQ: type of q and o; T: type of the products' operands.  fp16 rows against
// a cache (whose values need bf16's exponents) enter as two bf16 terms, and
// so do their probabilities.
template <typename TQ, typename T, int DP, typename KV>
__global__ __launch_bounds__(256) void attn_fwd_kernel(typename KV::Args args) {
    constexpr int NC = DP / 8, NS = DP / 32, ND = DP / 16, NT = sizeof(TQ) == sizeof(T) && __is_same(TQ, T) ? 1 : 2;
    typedef typename Vec<T>::x8 X8;
    typedef typename Vec<T>::x4 X4;
    typedef typename Vec<TQ>::x8 Q8;
    typedef typename Vec<TQ>::x4 Q4;
    __shared__ T sk[kBN * DP], sv[kBN * DP];
    __shared__ int s_in[KV::kHoles ? kBN : 1];

    const AttnArgs &a = KV::attn(args);
    const int item = xcd_item(blockIdx.x, a.per);
    if (item >= a.tiles * a.kv_heads) return;
    const int hkv = item / a.tiles;
    Seq s;
    if (!KV::find(args, item % a.tiles, s)) return;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
    const int row0 = s.tile * kBM, rows = s.q_len * a.group;
    const int wrow = row0 + wave * 32 + r;

    // this lane's rows: wrow and wrow + 16
    int pos[2];
    int64_t o_at[2], l_at[2];
    X8 qf[NT][2][NS];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int row = wrow + 16 * t;
        const bool in = row < rows;
        const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
        pos[t] = in ? tok + s.shift : -1;
        o_at[t] = in ? s.b * a.o_b + (s.q0 + tok) * a.o_t + h * a.o_h : -1;
        l_at[t] = s.b * a.lse_b + h * a.lse_h + s.q0 + tok;
        const TQ *qp = (const TQ *)a.q + s.b * a.q_b + (s.q0 + tok) * a.q_t + h * a.q_h;
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            const int c = st * 4 + g;
            const Q8 x = in && c * 8 < a.dim ? *(const Q8 *)(qp + c * 8) : Q8{};
            if constexpr (NT == 1)
                qf[0][t][st] = x;
            else
                split(x, qf[0][t][st], qf[1][t][st]);
        }
    }

    f32x4 o[ND][2];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d][0] = o[d][1] = f32x4{0, 0, 0, 0};

    // the keys that some row of the tile sees: the sinks, then [lo, hi)
    const int pmin = div_by(row0, a.by_group) + s.shift;
    const int pmax = div_by(min(row0 + kBM, rows) - 1, a.by_group) + s.shift;
    const int hi = min(pmax + 1, s.k_len), lo = a.window ? max(0, pmin - a.window + 1) : 0;
    const int t_sink = (min(a.sinks, hi) + kBN - 1) / kBN, t_hi = hi > 0 ? (hi + kBN - 1) / kBN : 0;
    const int t_lo = lo / kBN;
    auto next = [&](int t) { return t + 1 < t_sink ? t + 1 : max(t + 1, t_lo); };
    int t = t_sink > 0 ? 0 : t_lo;

    KV kv;
    kv.init(args, s, hkv);
    if (t < t_hi) kv.load(t * kBN);
    while (t < t_hi) {
        const int j0 = t * kBN, tn = next(t);
        __syncthreads();
        kv.store(sk, sv);
        if (KV::kHoles) {
            if constexpr (KV::kHoles)
                if (kv.part == 0) s_in[kv.row] = kv.in;
        }
        __syncthreads();
        if (tn < t_hi) kv.load(tn * kBN);

        f32x4 st[4][2];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            st[kt][0] = st[kt][1] = f32x4{0, 0, 0, 0};
            const int j = kt * 16 + r;
#pragma unroll
            for (int x = 0; x < NS; ++x) {
                const X8 kf = *(const X8 *)(sk + j * DP + swz<NC>(j, x * 4 + g) * 8);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    st[kt][0] = mfma(kf, qf[n][0][x], st[kt][0]);
                    st[kt][1] = mfma(kf, qf[n][1][x], st[kt][1]);
                }
            }
        }
        bool full = j0 + kBN - 1 <= pmin && (!a.window || j0 > pmax - a.window || j0 + kBN - 1 < a.sinks);
        if constexpr (KV::kHoles) full = full & __all(s_in[lane]);
        if (!full) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = j0 + kt * 16 + g * 4 + i;
                    bool in = true;
                    if constexpr (KV::kHoles) in = s_in[kt * 16 + g * 4 + i];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const bool see = in & sees(j, pos[x], window_low(pos[x], a.window), a.sinks);
                        st[kt][x][i] = see ? st[kt][x][i] : -INFINITY;
                    }
                }
        }
        X8 pf[NT][2][2];  // [term][pair of key tiles][row]
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float mx = m[x];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, st[kt][x][i]);
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            // a row that has seen nothing keeps -inf; its probabilities are 0
            const float mc = mx == -INFINITY ? 0.f : mx * a.c;
            const float alpha = __builtin_amdgcn_exp2f(m[x] * a.c - mc);
            m[x] = mx;
            float sum = 0.f;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kt][x][i], a.c, -mc));
                    sum += p;
                    // the probabilities are the product's operand in the
                    // inputs' type; their sum is of the unrounded ones
                    pf[0][kt >> 1][x][(kt & 1) * 4 + i] = (T)p;
                    if constexpr (NT == 2)
                        pf[1][kt >> 1][x][(kt & 1) * 4 + i] = (T)(p - (float)pf[0][kt >> 1][x][(kt & 1) * 4 + i]);
                }
            l[x] = l[x] * alpha + sum;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d][x] *= alpha;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int j = u * 32 + g * 4 + (r >> 2);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const int c = d * 2 + ((r & 3) >> 1), e = (r & 1) * 4;
                const X4 v0 = read_tr<T>(sv + j * DP + swz<NC>(j, c) * 8 + e);
                const X4 v1 = read_tr<T>(sv + (j + 16) * DP + swz<NC>(j + 16, c) * 8 + e);
                const X8 vf = join<X4, X8>(v0, v1);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    o[d][0] = mfma(vf, pf[n][u][0], o[d][0]);
                    o[d][1] = mfma(vf, pf[n][u][1], o[d][1]);
                }
            }
        }
        t = tn;
    }

#pragma unroll
    for (int x = 0; x < 2; ++x) {
        float sum = l[x] + __shfl_xor(l[x], 16);
        sum += __shfl_xor(sum, 32);
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        if (o_at[x] < 0) continue;
        TQ *op = (TQ *)a.o + o_at[x];
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            Q4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (TQ)(o[d][x][i] * inv);
            if (d * 16 + g * 4 < a.dim) *(Q4 *)(op + d * 16 + g * 4) = w;
        }
        if (a.lse && g == 0) a.lse[l_at[x]] = sum > 0.f ? m[x] * a.c + __log2f(sum) : sum != sum ? sum : -INFINITY;
    }
}

template <typename T>
hipError_t fwd(const AttnArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)a.per * 8);
    if (a.dim <= 64)
        attn_fwd_kernel<T, T, 64, DenseKV<T, 64>><<<grid, 256, 0, s>>>(a);
    else
        attn_fwd_kernel<T, T, 128, DenseKV<T, 128>><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

template <typename T>
hipError_t chunk(const AttendArgs &x, hipStream_t s) {
    const dim3 grid((unsigned)x.a.per * 8);
    if (x.p.dim == 64)
        attn_fwd_kernel<T, __bf16, 64, PagedKV<64>><<<grid, 256, 0, s>>>(x);
    else
        attn_fwd_kernel<T, __bf16, 128, PagedKV<128>><<<grid, 256, 0, s>>>(x);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_chunk(const AttendArgs &in, int dtype, hipStream_t s) {
    AttendArgs x = in;
    x.a.tiles = (int)(((int64_t)x.a.q_len * x.a.group + kBM - 1) / kBM) * x.a.batch;
    x.a.per = (int)(((int64_t)x.a.tiles * x.a.kv_heads + 7) / 8);
    return dtype == LSMX_BF16 ? chunk<__bf16>(x, s) : chunk<_Float16>(x, s);
}

hipError_t launch_attn_fwd(const AttnArgs &in, int dtype, hipStream_t s) {
    AttnArgs a = in;
    if (a.offsets)
        a.tiles = (int)(((int64_t)a.tokens * a.group + kBM - 1) / kBM) + a.batch + 2;
    else
        a.tiles = (int)(((int64_t)a.q_len * a.group + kBM - 1) / kBM) * a.batch;
    a.per = (int)(((int64_t)a.tiles * a.kv_heads + 7) / 8);
    return dtype == LSMX_BF16 ? fwd<__bf16>(a, s) : fwd<_Float16>(a, s);
}

}  // namespace lsmx
