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
#include "lsmx_dma.h"

namespace lsmx {
namespace {

constexpr int kBN = 64;  // keys of a tile

// Waits for a wave's own direct-to-LDS loads (issued in inline assembly, which
// the compiler does not count).
LSMX_DEV void wait_dma() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Keys and values as they lie in memory, loaded straight into LDS: lane l of
// a load fills 16-byte position l, so the swizzle is in the addresses.  The
// descriptor starts at the tile's first key; keys past the sequence and
// chunks past head_dim get an offset past its end and read zeros.
template <typename T, int DP, int NW>
struct DenseKV {
    static constexpr int NC = DP / 8, NU = kBN * NC / 64 / NW;  // loads of a wave, each of K and V
    static constexpr bool kHoles = false;
    typedef AttnArgs Args;
    const T *k, *v;
    int64_t k_t, v_t;
    int k_len;
    uint32_t row, chunk;  // of lane's first load; the others are NW * 64 / NC rows on
    bool in;

    LSMX_DEV static const AttnArgs &attn(const Args &a) { return a; }
    LSMX_DEV static bool find(const Args &a, int t, int size, Seq &s) {
        // the last tile of a sequence first: under a causal mask it is the longest
        return find_tile(a, a.tiles - 1 - t, size, a.group, a.q_len, s);
    }
    LSMX_DEV void init(const AttnArgs &a, const Seq &s, int hkv) {
        k = (const T *)a.k + s.b * a.k_b + s.k0 * a.k_t + hkv * a.k_h;
        v = (const T *)a.v + s.b * a.v_b + s.k0 * a.v_t + hkv * a.v_h;
        k_t = a.k_t, v_t = a.v_t, k_len = s.k_len;
    }
    LSMX_DEV void fetch(int j0, T *sk, T *sv, int dim) {
        const v4i_rsrc rk = buf_rsrc(k + j0 * k_t, 0x7FFFFFFF), rv = buf_rsrc(v + j0 * v_t, 0x7FFFFFFF);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
        const uint32_t bk = lds_u32(sk), bv = lds_u32(sv);
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int at = (u * NW + wave) * 64, j = (at + lane) / NC, c = swz<NC>(j, lane % NC);
            const bool ok = j0 + j < k_len && c * 8 < dim;
            dma_x4(ok ? (uint32_t)(j * (int)k_t + c * 8) * 2 : 0x80000000u, rk, bk + at * 16);
            dma_x4(ok ? (uint32_t)(j * (int)v_t + c * 8) * 2 : 0x80000000u, rv, bv + at * 16);
        }
    }
    LSMX_DEV void land(T *, T *, int *) { wait_dma(); }
};

// Keys and values of a paged MXFP4 cache, expanded to bf16 on their way into
// LDS (exact).  Four threads take a key's vector, and (the same four of 4
// waves, the next of 8) a value's.
template <int DP, int NW>
struct PagedKV {
    static constexpr int NC = DP / 8, NQ = DP / 32;  // words of codes of a thread
    static constexpr bool kHoles = true, kBoth = NW == 4;
    typedef AttendArgs Args;
    typedef __bf16 T;
    const Pool *p;
    int b, h, k_len, row, part;
    uint32_t kr[NQ], vr[NQ];
    uint32_t ke, ve;
    bool in, is_v;

    LSMX_DEV static const AttnArgs &attn(const Args &a) { return a.a; }
    LSMX_DEV static bool find(const Args &x, int t, int size, Seq &s) {
        const AttnArgs &a = x.a;
        const int per = (a.q_len * a.group + size - 1) / size;
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
        p = &a.p, b = s.b, h = hkv, k_len = s.k_len;
        row = (threadIdx.x & 255) >> 2, part = threadIdx.x & 3, is_v = threadIdx.x >= 256;
    }
    LSMX_DEV static void codes(uint32_t (&w)[NQ], const uint8_t *c) {
        if constexpr (NQ == 4)
            *(u32x4 *)w = *(const u32x4 *)c;
        else
            *(u32x2 *)w = *(const u32x2 *)c;
    }
    LSMX_DEV void fetch(int j0, T *, T *, int) {
        const int j = j0 + row, pg = j < k_len ? p->page_of(b, j) : -1;
        in = pg >= 0;
#pragma unroll
        for (int i = 0; i < NQ; ++i) kr[i] = vr[i] = 0;
        ke = ve = 0;
        if (in) {
            const int64_t v = p->vec(pg, h, j);
            const int blk = part * (DP / 32) / 4;
            codes(kr, (is_v ? p->vc : p->kc) + v * (DP / 2) + part * (DP / 8));
            ke = (is_v ? p->vs : p->ks)[v * (DP / 32) + blk];
            if constexpr (kBoth) {
                codes(vr, p->vc + v * (DP / 2) + part * (DP / 8));
                ve = p->vs[v * (DP / 32) + blk];
            }
        }
    }
    LSMX_DEV void land(T *sk, T *sv, int *s_in) {
        const float ksc = e8m0_to_f32(ke), vsc = e8m0_to_f32(ve);
        T *first = is_v ? sv : sk;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int c = swz<NC>(row, part * NQ + i);
            *(bf16x8 *)(first + row * DP + c * 8) = fp4x8_to_bf16(kr[i], ksc);
            if constexpr (kBoth) *(bf16x8 *)(sv + row * DP + c * 8) = fp4x8_to_bf16(vr[i], vsc);
        }
        if (part == 0 && !is_v) s_in[row] = in;
    }
};

// NW waves of RT x 16 rows.  TQ: type of q and o; T: type of the products'
// operands.  fp16 rows against a cache (whose values need bf16's exponents)
// enter as two bf16 terms, and so do their probabilities.
template <typename TQ, typename T, int DP, int RT, int NW, typename KV>
__global__ __launch_bounds__(NW * 64, 2) void attn_fwd_kernel(typename KV::Args args) {
    constexpr int NC = DP / 8, NS = DP / 32, ND = DP / 16, NT = __is_same(TQ, T) ? 1 : 2, BM = NW * RT * 16;
    // a row's maximum is followed only when it grows by this factor 2^8: the
    // probabilities stay below 2^8 and O is rescaled a few times per row
    constexpr float kLazy = 8.f;
    typedef typename Vec<T>::x8 X8;
    typedef typename Vec<T>::x4 X4;
    typedef typename Vec<TQ>::x8 Q8;
    typedef typename Vec<TQ>::x4 Q4;
    __shared__ __attribute__((aligned(16))) T sk[2][kBN * DP], sv[2][kBN * DP];
    __shared__ int s_in[2][KV::kHoles ? kBN : 1];

    const AttnArgs &a = KV::attn(args);
    const int item = xcd_item(blockIdx.x, a.per);
    if (item >= a.tiles * a.kv_heads) return;
    const int hkv = item / a.tiles;
    Seq s;
    if (!KV::find(args, item % a.tiles, BM, s)) return;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, r = lane & 15;
    const int row0 = s.tile * BM, rows = s.q_len * a.group, wrow0 = row0 + wave * RT * 16;

    // the keys that some row of the tile sees: the sinks, then [lo, hi)
    const int pmin = div_by(row0, a.by_group) + s.shift;
    const int pmax = div_by(min(row0 + BM, rows) - 1, a.by_group) + s.shift;
    const int hi = min(pmax + 1, s.k_len), lo = a.window ? max(0, pmin - a.window + 1) : 0;
    const int t_sink = (min(a.sinks, hi) + kBN - 1) / kBN, t_hi = hi > 0 ? (hi + kBN - 1) / kBN : 0;
    const int t_lo = lo / kBN;
    auto next = [&](int t) { return t + 1 < t_sink ? t + 1 : max(t + 1, t_lo); };
    int t = t_sink > 0 ? 0 : t_lo, buf = 0;
    // and those of this wave's rows
    const int wmin = div_by(min(wrow0, rows - 1), a.by_group) + s.shift;
    const int wmax = wrow0 < rows ? div_by(min(wrow0 + RT * 16, rows) - 1, a.by_group) + s.shift : -1;

    KV kv;
    kv.init(args, s, hkv);
    if (t < t_hi) kv.fetch(t * kBN, sk[0], sv[0], a.dim);

    // this lane's rows: wrow0 + r + 16 x
    int pos[RT], low[RT];
    X8 qf[NT][RT][NS];
#pragma unroll
    for (int x = 0; x < RT; ++x) {
        const int row = wrow0 + r + 16 * x;
        const bool in = row < rows;
        const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
        pos[x] = in ? tok + s.shift : -1;
        low[x] = window_low(pos[x], a.window);
        const TQ *qp = (const TQ *)a.q + s.b * a.q_b + (s.q0 + tok) * a.q_t + h * a.q_h;
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            const int c = st * 4 + g;
            const Q8 w = in && c * 8 < a.dim ? *(const Q8 *)(qp + c * 8) : Q8{};
            if constexpr (NT == 1)
                qf[0][x][st] = w;
            else
                split(w, qf[0][x][st], qf[1][x][st]);
        }
    }

    f32x4 o[ND][RT];
    float m[RT], l[RT];
#pragma unroll
    for (int x = 0; x < RT; ++x) {
        m[x] = -INFINITY, l[x] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d][x] = f32x4{0, 0, 0, 0};
    }
    const float lazy = kLazy / a.c;

    if (t < t_hi) kv.land(sk[0], sv[0], s_in[0]);
    __syncthreads();
    while (t < t_hi) {
        const int j0 = t * kBN, tn = next(t);
        if (tn < t_hi) kv.fetch(tn * kBN, sk[buf ^ 1], sv[buf ^ 1], a.dim);
        // hidden from every row of the wave: nothing to do
        const bool none = j0 > wmax || (a.window && j0 + kBN - 1 <= wmin - a.window && j0 >= a.sinks);
        if (!none) {
            const T *ck = sk[buf], *cv = sv[buf];
            f32x4 st[4][RT];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                const int j = kt * 16 + r;
#pragma unroll
                for (int x = 0; x < RT; ++x) st[kt][x] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int y = 0; y < NS; ++y) {
                    const X8 kf = *(const X8 *)(ck + j * DP + swz<NC>(j, y * 4 + g) * 8);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int x = 0; x < RT; ++x) st[kt][x] = mfma(kf, qf[n][x][y], st[kt][x]);
                }
            }
            bool full = j0 + kBN - 1 <= wmin && (!a.window || j0 > wmax - a.window || j0 + kBN - 1 < a.sinks);
            if constexpr (KV::kHoles) full = full & __all(s_in[buf][lane]);
            if (!full) {
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = j0 + kt * 16 + g * 4 + i;
                        bool in = true;
                        if constexpr (KV::kHoles) in = s_in[buf][kt * 16 + g * 4 + i];
#pragma unroll
                        for (int x = 0; x < RT; ++x) {
                            const bool see = in & sees(j, pos[x], low[x], a.sinks);
                            st[kt][x][i] = see ? st[kt][x][i] : -INFINITY;
                        }
                    }
            }
            float mx[RT];
            bool grow = false;
#pragma unroll
            for (int x = 0; x < RT; ++x) {
                mx[x] = st[0][x][0];
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx[x] = fmaxf(mx[x], st[kt][x][i]);
                mx[x] = fmaxf(mx[x], __shfl_xor(mx[x], 16));
                mx[x] = fmaxf(mx[x], __shfl_xor(mx[x], 32));
                grow = grow | (mx[x] > m[x] + lazy);
            }
            if (__any(grow)) {
#pragma unroll
                for (int x = 0; x < RT; ++x) {
                    const float top = fmaxf(m[x], mx[x]);
                    // a row that has seen nothing keeps -inf and its zeros
                    const float alpha = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[x] - top) * a.c);
                    m[x] = top;
                    l[x] *= alpha;
#pragma unroll
                    for (int d = 0; d < ND; ++d) o[d][x] *= alpha;
                }
            }
            X8 pf[NT][2][RT];  // [term][pair of key tiles][row]
#pragma unroll
            for (int x = 0; x < RT; ++x) {
                const float mc = m[x] == -INFINITY ? 0.f : m[x] * a.c;
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
                l[x] += sum;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int j = u * 32 + g * 4 + (r >> 2);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const int c = d * 2 + ((r & 3) >> 1), e = (r & 1) * 4;
                    const X4 v0 = read_tr<T>(cv + j * DP + swz<NC>(j, c) * 8 + e);
                    const X4 v1 = read_tr<T>(cv + (j + 16) * DP + swz<NC>(j + 16, c) * 8 + e);
                    const X8 vf = join<X4, X8>(v0, v1);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int x = 0; x < RT; ++x) o[d][x] = mfma(vf, pf[n][u][x], o[d][x]);
                }
            }
        }
        buf ^= 1;
        if (tn < t_hi) kv.land(sk[buf], sv[buf], s_in[buf]);
        __syncthreads();
        t = tn;
    }

#pragma unroll
    for (int x = 0; x < RT; ++x) {
        float sum = l[x] + __shfl_xor(l[x], 16);
        sum += __shfl_xor(sum, 32);
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        const int row = wrow0 + r + 16 * x;
        if (row >= rows) continue;
        const int tok = div_by(row, a.by_group), h = hkv * a.group + row - tok * a.group;
        TQ *op = (TQ *)a.o + s.b * a.o_b + (s.q0 + tok) * a.o_t + h * a.o_h;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            Q4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (TQ)(o[d][x][i] * inv);
            if (d * 16 + g * 4 < a.dim) *(Q4 *)(op + d * 16 + g * 4) = w;
        }
        if (a.lse && g == 0)
            a.lse[s.b * a.lse_b + h * a.lse_h + s.q0 + tok] =
                sum > 0.f ? m[x] * a.c + __log2f(sum) : sum != sum ? sum : -INFINITY;
    }
}

// Row tiles over all sequences, and the grid of their items over 8 XCDs.
void tiles_of(AttnArgs &a, int rows) {
    if (a.offsets)
        a.tiles = (int)(((int64_t)a.tokens * a.group + rows - 1) / rows) + a.batch + 2;
    else
        a.tiles = (int)(((int64_t)a.q_len * a.group + rows - 1) / rows) * a.batch;
    a.per = (int)(((int64_t)a.tiles * a.kv_heads + 7) / 8);
}

// 8 waves share the keys in LDS where their tiles still give each CU two
// workgroups' worth of rows; else 4 waves.
bool wide(const AttnArgs &a, int rows8) {
    const int64_t rows = (int64_t)(a.offsets ? a.tokens : a.q_len) * a.group * (a.offsets ? 1 : a.batch);
    return rows * a.kv_heads >= (int64_t)512 * rows8;
}

template <typename T, int DP, int RT>
hipError_t fwd(AttnArgs a, hipStream_t s) {
    if (wide(a, 8 * RT * 16)) {
        tiles_of(a, 8 * RT * 16);
        attn_fwd_kernel<T, T, DP, RT, 8, DenseKV<T, DP, 8>><<<(unsigned)a.per * 8, 512, 0, s>>>(a);
    } else {
        tiles_of(a, 4 * RT * 16);
        attn_fwd_kernel<T, T, DP, RT, 4, DenseKV<T, DP, 4>><<<(unsigned)a.per * 8, 256, 0, s>>>(a);
    }
    return hipGetLastError();
}

template <typename T, int DP>
hipError_t chunk(AttendArgs x, hipStream_t s) {
    if (wide(x.a, 256)) {
        tiles_of(x.a, 256);
        attn_fwd_kernel<T, __bf16, DP, 2, 8, PagedKV<DP, 8>><<<(unsigned)x.a.per * 8, 512, 0, s>>>(x);
    } else {
        tiles_of(x.a, 128);
        attn_fwd_kernel<T, __bf16, DP, 2, 4, PagedKV<DP, 4>><<<(unsigned)x.a.per * 8, 256, 0, s>>>(x);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_chunk(const AttendArgs &x, int dtype, hipStream_t s) {
    if (dtype == LSMX_BF16) return x.p.dim == 64 ? chunk<__bf16, 64>(x, s) : chunk<__bf16, 128>(x, s);
    return x.p.dim == 64 ? chunk<_Float16, 64>(x, s) : chunk<_Float16, 128>(x, s);
}

hipError_t launch_attn_fwd(const AttnArgs &a, int dtype, hipStream_t s) {
    if (dtype == LSMX_BF16) return a.dim <= 64 ? fwd<__bf16, 64, 2>(a, s) : fwd<__bf16, 128, 2>(a, s);
    return a.dim <= 64 ? fwd<_Float16, 64, 2>(a, s) : fwd<_Float16, 128, 2>(a, s);
}

}  // namespace lsmx
