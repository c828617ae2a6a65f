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

// Keys and values as they lie in memory, loaded straight into LDS: lane l of
// a load fills 16-byte position l, so the swizzle is in the addresses.  The
// descriptor starts at the tile's first key; keys past the sequence and
// chunks past head_dim get an offset past its end and read zeros.
template <typename T, int DP, int NW>
struct DenseKV {
    static constexpr int NC = DP / 8, NU = kBN * NC / 64 / NW;  // loads of a wave, each of K and V
    static constexpr bool kHoles = false;
    typedef AttnArgs Args;
    LSMX_DEV static int splits(const Args &) { return 1; }
    const T *k, *v;
    int64_t k_t, v_t;
    int k_len;

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
    LSMX_DEV void fetch(const T *x, int64_t x_t, int j0, T *to, int dim) {
        const v4i_rsrc rs = buf_rsrc(x + j0 * x_t, 0x7FFFFFFF);
        const int wave = uniform((threadIdx.x >> 6) % NW), lane = threadIdx.x & 63;
        const uint32_t lds = lds_u32(to);
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int at = (u * NW + wave) * 64, j = (at + lane) / NC, c = swz<NC>(j, lane % NC);
            const bool ok = j0 + j < k_len && c * 8 < dim;
            dma_x4(ok ? (uint32_t)(j * (int)x_t + c * 8) * 2 : 0x80000000u, rs, lds + at * 16);
        }
    }
    LSMX_DEV void fetch(int j0, int, int, T *sk, T *sv, int *, int dim) {
        fetch(k, k_t, j0, sk, dim);
        fetch(v, v_t, j0, sv, dim);
    }
    LSMX_DEV void start(int j0, int, int, T *sk, T *sv, int *, int dim) { fetch(j0, 0, 0, sk, sv, nullptr, dim); }
    LSMX_DEV void land() { wait_dma(); }
};

// Keys and values of a paged MXFP4 cache, expanded to the rows' type on their way into
// LDS.  Four of the 256 threads take a key's vector, and a value's.
template <typename T, int DP>
struct PagedKV {
    static constexpr int NC = DP / 8, NQ = DP / 32;  // words of codes of a thread
    static constexpr bool kHoles = true;
    typedef AttendArgs Args;
    LSMX_DEV static int splits(const Args &a) { return a.splits; }
    const Pool *p;
    int b, h, k_len, row, part;
    uint32_t kr[NQ], vr[NQ];
    uint32_t ke, ve;
    int pg, pgn;  // page of the codes in registers, and of the next tile's
    bool bad;     // there were blocks that T does not hold

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
        p = &a.p, b = s.b, h = hkv, k_len = s.k_len, row = (threadIdx.x & 255) >> 2, part = threadIdx.x & 3, bad = false;
    }
    LSMX_DEV int page(int j0) const {
        const int j = j0 + row;
        return j0 >= 0 && j < k_len ? p->page_of(b, j) : -1;
    }
    // this thread's part of vector j
    LSMX_DEV void codes(int j, const uint8_t *codes, const uint8_t *scale, uint32_t (&w)[NQ], uint32_t &e) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) w[i] = 0;
        e = 127;
        if (pg >= 0) {
            const int64_t v = p->vec(pg, h, j);
            const uint8_t *c = codes + v * (DP / 2) + part * (DP / 8);
            if constexpr (NQ == 4)
                *(u32x4 *)w = *(const u32x4 *)c;
            else
                *(u32x2 *)w = *(const u32x2 *)c;
            e = scale[v * (DP / 32) + part * (DP / 32) / 4];
        }
    }
    LSMX_DEV void store(T *to, const uint32_t (&w)[NQ], uint32_t e) {
        const float sc = block_scale<T>(e);
        bad = bad | !holds<T>(e);
#pragma unroll
        for (int i = 0; i < NQ; ++i)
            *(typename Vec<T>::x8 *)(to + row * DP + swz<NC>(row, part * NQ + i) * 8) = fp4x8<T>(w[i], sc);
    }
    // The first tile j0 (next j1, then j2; -1: none) into LDS, the next one's
    // codes on their way.
    LSMX_DEV void start(int j0, int j1, int j2, T *sk, T *sv, int *s_in, int) {
        pg = page(j0), pgn = page(j1);
        load(j0);
        fetch(j0, j1, j2, sk, sv, s_in, 0);
    }
    LSMX_DEV void load(int j0) {
        codes(j0 + row, p->kc, p->ks, kr, ke);
        codes(j0 + row, p->vc, p->vs, vr, ve);
    }
    // Tile j0, whose codes are in registers, into LDS; those of j1 on their
    // way, and the page of j2: each load has a round to land.
    LSMX_DEV void fetch(int j0, int j1, int j2, T *sk, T *sv, int *s_in, int) {
        store(sk, kr, ke);
        store(sv, vr, ve);
        if (part == 0) s_in[row] = pg >= 0;
        pg = pgn;
        load(j1);
        pgn = page(j2);
    }
    LSMX_DEV void land() {}
};

// KS groups (each with its share of the keys) of NW waves of RT x 16 rows.
//
// The loop is pipelined over two key tiles: the scores of the next tile are
// products that do not wait for anything, and stand between the exponentials
// of this one, which are as much work for the vector unit as both products
// are for the matrix unit.
//
// Bound by what a wave waits for and the few others cannot fill: the vector unit
// (exponentials, sums and conversions) is busy 58% of the cycles at head 128, the
// matrix unit 30%, neither ever full.  Waves per SIMD count: 2 at head 128, 3 at 64
// (registers allow it only while a step is 32 keys).  2 x 4096 tokens, 32/8 heads of
// 128, window 1024: 174 us a call = 694 TFLOP/s of the visible pairs (with the
// remainders of o stored for the backward 216 to 228); 16384 tokens of 8/1 heads
// of 64 through a window of 4096: 191 us = 631 TFLOP/s (1024 almost equal workgroups, of
// which 768 run at a time).  Heads of 72 to 120 take all products of 128, their
// chunks past the head are zeros: 4096 causal tokens of 32/8 heads of 80 171 us, 128 176.
template <typename T, int DP, int RT, int NW, int KS, typename KV>
__global__ __launch_bounds__(NW * KS * 64, DP == 128 ? 2 : KV::kHoles ? 4 : 3) void attn_fwd_kernel(typename KV::Args args) {
    constexpr int NC = DP / 8, NS = DP / 32, ND = DP / 16, BM = NW * RT * 16;
    // a row's maximum is followed only when it grows by a factor of 2^8 (fp16:
    // 2^4, below its range with the lift): O is rescaled a few times per row
    constexpr float kLazy = kLift<T> > 0.f ? 4.f : 8.f;
    typedef typename Vec<T>::x8 X8;
    typedef typename Vec<T>::x4 X4;
    __shared__ __attribute__((aligned(16))) T s_kv[KS][2][2][kBN * DP];  // [group][keys, values][buffer]
    __shared__ int s_held[KS][2][KV::kHoles ? kBN : 1];

    const AttnArgs &a = KV::attn(args);
    const int splits = KV::splits(args);
    const Item item = item_of(a, splits);
    const int hkv = item.head, share = item.share;
    if (hkv >= a.kv_heads) return;
    Seq s;
    if (!KV::find(args, item.tile, BM, s)) return;

    const int lane = threadIdx.x & 63, wave = uniform((threadIdx.x >> 6) % NW), g = lane >> 4, r = lane & 15;
    const int group = KS == 1 ? 0 : uniform(threadIdx.x / (NW * 64));
    T(&sk)[2][kBN * DP] = s_kv[group][0], (&sv)[2][kBN * DP] = s_kv[group][1];
    auto &s_in = s_held[group];
    const int row0 = s.tile * BM, rows = s.q_len * a.group, wrow0 = row0 + wave * RT * 16;

    // the keys that some row of the tile sees: the sinks, then [lo, hi)
    const int pmin = div_by(row0, a.by_group) + s.shift;
    const int pmax = div_by(min(row0 + BM, rows) - 1, a.by_group) + s.shift;
    const int hi = min(pmax + 1, s.k_len), lo = a.window ? max(0, pmin - a.window + 1) : 0;
    const int t_sink = (min(a.sinks, hi) + kBN - 1) / kBN, t_hi = hi > 0 ? (hi + kBN - 1) / kBN : 0;
    const int t_lo = max(lo / kBN, t_sink), nt = t_sink + max(0, t_hi - t_lo);
    const int first = (int)((int64_t)nt * share / splits), last = (int)((int64_t)nt * (share + 1) / splits);
    const int rounds = (last - first + KS - 1) / KS;
    // first key of the group's tile of round k, -1 past the last
    auto start_of = [&](int k) {
        const int i = first + k * KS + group;
        return i < last ? (i < t_sink ? i : t_lo + i - t_sink) * kBN : -1;
    };
    // and the positions of this wave's rows
    const int wmin = div_by(min(wrow0, rows - 1), a.by_group) + s.shift;
    const int wmax = div_by(min(wrow0 + RT * 16, rows) - 1, a.by_group) + s.shift;

    KV kv;
    kv.init(args, s, hkv);
    int j0 = start_of(0);
    if (j0 >= 0) kv.start(j0, start_of(1), start_of(2), sk[0], sv[0], s_in[0], a.dim);

    // this lane's rows: wrow0 + r + 16 x
    int pos[RT], low[RT];
    X8 qf[RT][NS];
#pragma unroll
    for (int x = 0; x < RT; ++x) {
        const int row = wrow0 + r + 16 * x;
        const bool in = row < rows;
        const int tok = div_by(in ? row : 0, a.by_group), h = hkv * a.group + (in ? row : 0) - tok * a.group;
        pos[x] = in ? tok + s.shift : -1;
        low[x] = window_low(pos[x], a.window);
        const T *qp = (const T *)a.q + s.b * a.q_b + (s.q0 + tok) * a.q_t + h * a.q_h;
#pragma unroll
        for (int st = 0; st < NS; ++st) {
            const int c = st * 4 + g;
            qf[x][st] = in && c * 8 < a.dim ? *(const X8 *)(qp + c * 8) : X8{};
        }
    }

    f32x4 o[ND][RT], st[2][RT];
    // of each row: maximum, its limit, times c; sum over this lane's keys
    float m[RT], limit[RT], mc[RT], l[RT];
#pragma unroll
    for (int x = 0; x < RT; ++x) {
        m[x] = limit[x] = -INFINITY, mc[x] = l[x] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d][x] = f32x4{0, 0, 0, 0};
    }
    const float lazy = kLazy / a.c;

    // scores of 32 keys from row j0 of a tile on
    // (lr: r, opaque where the lane's places in LDS are made anew each time;
    // held over the loop they would not fit the registers)
    auto scores = [&](const T *ck, int j0, int lr, f32x4 (&z)[2][RT]) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const int j = j0 + kt * 16 + lr;
#pragma unroll
            for (int x = 0; x < RT; ++x) z[kt][x] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int y = 0; y < NS; ++y) {
                const X8 kf = *(const X8 *)(ck + j * DP + swz<NC>(j, y * 4 + g) * 8);
#pragma unroll
                for (int x = 0; x < RT; ++x) z[kt][x] = mfma(kf, qf[x][y], z[kt][x]);
            }
        }
    };
    // those that a row does not see, to -inf
    auto hide = [&](int j0, const int *held, f32x4 (&z)[2][RT]) {
        bool full = j0 + 31 <= wmin && (!a.window || j0 > wmax - a.window || j0 + 31 < a.sinks);
        if constexpr (KV::kHoles) full = full & __all(held[lane & 31]);
        if (full) return;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = j0 + kt * 16 + g * 4 + i;
                bool in = true;
                if constexpr (KV::kHoles) in = held[kt * 16 + g * 4 + i];
#pragma unroll
                for (int x = 0; x < RT; ++x) {
                    const bool see = in & sees(j, pos[x], low[x], a.sinks);
                    z[kt][x][i] = see ? z[kt][x][i] : -INFINITY;
                }
            }
    };
    // 32 keys whose scores are in st, with their values from row jv of cv on;
    // the scores of the 32 from row jk of ck on, if there are more, take their place
    auto step = [&](auto more, const T *ck, int jk, const T *cv, int jv) {
        constexpr bool kMore = decltype(more)::value;
        float mx[RT];
        bool grow = false;
#pragma unroll
        for (int x = 0; x < RT; ++x) {
            mx[x] = fmaxf(fmaxf(st[0][x][0], st[0][x][1]), st[0][x][2]);
            mx[x] = fmaxf(fmaxf(mx[x], st[0][x][3]), st[1][x][0]);
            mx[x] = fmaxf(fmaxf(mx[x], st[1][x][1]), st[1][x][2]);
            mx[x] = fmaxf(mx[x], st[1][x][3]);
            grow = grow | (mx[x] > limit[x]);
        }
        // the row's maximum over its 4 lanes is only needed when it grows
        if (__any(grow)) {
#pragma unroll
            for (int x = 0; x < RT; ++x) {
                const float top = fmaxf(m[x], max_rows(mx[x]));
                // a row that has seen nothing keeps -inf and its zeros
                const float alpha = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[x] - top) * a.c);
                m[x] = top;
                limit[x] = top + lazy;
                mc[x] = top == -INFINITY ? 0.f : top * a.c - kLift<T>;
                l[x] *= alpha;
#pragma unroll
                for (int d = 0; d < ND; ++d) o[d][x] *= alpha;
            }
        }
        int lr = r;
        if constexpr (DP == 128 && !KV::kHoles) asm volatile("" : "+v"(lr));
        X8 vf[ND];
        const int j = jv + g * 4 + (lr >> 2);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const int c = d * 2 + ((lr & 3) >> 1), e = (lr & 1) * 4;
            vf[d] = join<X4, X8>(read_tr<T>(cv + j * DP + swz<NC>(j, c) * 8 + e),
                                 read_tr<T>(cv + (j + 16) * DP + swz<NC>(j + 16, c) * 8 + e));
        }
        f32x4 zn[2][RT];
        if constexpr (kMore) scores(ck, jk, lr, zn);
        X8 pf[RT];
#pragma unroll
        for (int x = 0; x < RT; ++x) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kt][x][i], a.c, -mc[x]));
                    l[x] += p;
                    // the probabilities are the product's operand in the
                    // inputs' type; their sum is of the unrounded ones
                    pf[x][kt * 4 + i] = (T)p;
                }
        }
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int x = 0; x < RT; ++x) o[d][x] = mfma(vf[d], pf[x], o[d][x]);
        if constexpr (kMore) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int x = 0; x < RT; ++x) st[kt][x] = zn[kt][x];
        }
    };

    wait_dma();
    __syncthreads();
    if (j0 >= 0) {
        scores(sk[0], 0, r, st);
        hide(j0, s_in[0], st);
    }
    int n = 0;  // the round's tile is in buffer n
    for (int k = 0; k < rounds; ++k) {
        const int j1 = start_of(k + 1);
        if (j1 >= 0) kv.fetch(j1, start_of(k + 2), start_of(k + 3), sk[n ^ 1], sv[n ^ 1], s_in[n ^ 1], a.dim);
        if (j0 >= 0) {
            step(BoolC<true>{}, sk[n], 32, sv[n], 0);
            hide(j0 + 32, s_in[n] + (KV::kHoles ? 32 : 0), st);
        }
        if (j1 >= 0) kv.land();
        if (k + 1 < rounds) __syncthreads();
        if (j1 >= 0) {
            step(BoolC<true>{}, sk[n ^ 1], 0, sv[n], 32);
            hide(j1, s_in[n ^ 1], st);
        } else if (j0 >= 0) {
            step(BoolC<false>{}, sk[0], 0, sv[n], 32);
        }
        if (k + 1 < rounds) __syncthreads();
        n ^= 1, j0 = j1;
    }

    if constexpr (KV::kHoles && __is_same(T, _Float16)) {
        if (uniform(__syncthreads_or(kv.bad))) {
            attend_exact<T, DP, kBN>(args, s.b, hkv, share, row0, min(row0 + BM, rows), last - first,
                                     [=](int i) { return (first + i < t_sink ? first + i : t_lo + first + i - t_sink) * kBN; });
            return;
        }
    }
    if constexpr (KS == 2) {
        // the second group's sums through LDS to the first, which writes
        static_assert(NW * 64 * RT * ND * 16 + NW * 64 * RT * 8 <= sizeof(s_kv), "");
        float *x_o = (float *)&s_kv, *x_m = x_o + NW * 64 * RT * ND * 4;
        const int me = wave * 64 + lane;
        __syncthreads();
        if (group == 1) {
#pragma unroll
            for (int x = 0; x < RT; ++x) {
#pragma unroll
                for (int d = 0; d < ND; ++d) *(f32x4 *)(x_o + ((x * ND + d) * NW * 64 + me) * 4) = o[d][x];
                x_m[(x * 2) * NW * 64 + me] = m[x], x_m[(x * 2 + 1) * NW * 64 + me] = l[x];
            }
        }
        __syncthreads();
        if (group == 1) return;
#pragma unroll
        for (int x = 0; x < RT; ++x) {
            const float m2 = x_m[(x * 2) * NW * 64 + me], l2 = x_m[(x * 2 + 1) * NW * 64 + me], top = fmaxf(m[x], m2);
            const float f1 = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[x] - top) * a.c);
            const float f2 = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m2 - top) * a.c);
            m[x] = top;
            l[x] = l[x] * f1 + l2 * f2;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d][x] = o[d][x] * f1 + *(f32x4 *)(x_o + ((x * ND + d) * NW * 64 + me) * 4) * f2;
        }
    }

#pragma unroll
    for (int x = 0; x < RT; ++x) {
        const float sum = sum_rows(l[x]);
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        const int row = wrow0 + r + 16 * x;
        if (row >= rows) continue;
        if constexpr (KV::kHoles) {
            if (splits > 1) {
                const int64_t at = ((int64_t)(s.b * a.kv_heads + hkv) * splits + share) * rows + row;
#pragma unroll
                for (int d = 0; d < ND; ++d) *(f32x4 *)(args.part + at * DP + d * 16 + g * 4) = o[d][x];
                if (g == 0) args.part_m[at * 2] = m[x], args.part_m[at * 2 + 1] = sum;
                continue;
            }
        }
        const int tok = div_by(row, a.by_group), h = hkv * a.group + row - tok * a.group;
        const int64_t o_at = s.b * a.o_b + (s.q0 + tok) * a.o_t + h * a.o_h;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            X4 w, rest;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = o[d][x][i] * inv;
                w[i] = (T)f;
                rest[i] = (T)(f - (float)w[i]);
            }
            if (d * 16 + g * 4 < a.dim) {
                *(X4 *)((T *)a.o + o_at + d * 16 + g * 4) = w;
                if (a.o_lo) *(X4 *)((T *)a.o_lo + o_at + d * 16 + g * 4) = rest;
            }
        }
        if (a.lse && g == 0)
            a.lse[s.b * a.lse_b + h * a.lse_h + s.q0 + tok] =
                sum > 0.f ? m[x] * a.c - kLift<T> + __log2f(sum) : sum != sum ? sum : -INFINITY;
    }
}

// Row tiles over all sequences; the grid of their items.
unsigned tiles_of(AttnArgs &a, int rows, int splits = 1) {
    if (a.offsets)
        a.tiles = (int)(((int64_t)a.tokens * a.group + rows - 1) / rows) + a.batch + 2;
    else
        a.tiles = (int)(((int64_t)a.q_len * a.group + rows - 1) / rows) * a.batch;
    return order_items(a, (int64_t)a.tiles * a.kv_heads * splits);
}

// Workgroups of 4 waves: two or three of them on a CU run out of step, and one's
// products fall into another's exponentials.  (8 waves that share their tiles
// were in step: 201 against 179 us at 2 x 4096 tokens, 32/8 heads of 128.)
//
// A wave of 32 rows (kWide) reads half as much of LDS per product as one of 16
// (kNarrow), and is the faster when the rows give every SIMD as many as it
// holds: 2 at head 128, 3 at 64.  With fewer rows twice as many waves are, and
// below 2048 waves of 16 (two to a SIMD) the keys in two halves, each with 4
// waves of the workgroup.  T tokens, causal, 32/8 heads, us:
//             T    256    512   1024   1792   2560
//   wide     64    9.7   14.9   25.1   39.8   54.4    128   13.3  20.9  36.6  58.7  80.9
//   narrow         7.7   11.9   20.1   32.3   46.4           9.8  15.3  27.3  53.8  95.9
//   halves         7.0    9.7   16.1   34.1   54.5           9.1  13.0  26.2  64.2 119.7
// 16384 tokens of 8/1 heads of 64 through a window of 4096: wide 252, narrow 275.
enum Form { kWide, kNarrow, kHalves };
constexpr int kSimds = 1024;
Form form_of(const AttnArgs &a) {
    const int64_t waves = (int64_t)(a.offsets ? a.tokens : a.q_len) * a.group * (a.offsets ? 1 : a.batch) * a.kv_heads / 16;
    return waves >= (a.dim <= 64 ? 6 : 4) * kSimds ? kWide : waves > 2 * kSimds ? kNarrow : kHalves;
}

template <typename T, int DP>
hipError_t fwd(AttnArgs a, hipStream_t s) {
    const Form f = form_of(a);
    const unsigned grid = tiles_of(a, f == kWide ? 128 : 64);
    if (f == kWide)
        attn_fwd_kernel<T, DP, 2, 4, 1, DenseKV<T, DP, 4>><<<grid, 256, 0, s>>>(a);
    else if (f == kNarrow)
        attn_fwd_kernel<T, DP, 1, 4, 1, DenseKV<T, DP, 4>><<<grid, 256, 0, s>>>(a);
    else
        attn_fwd_kernel<T, DP, 1, 4, 2, DenseKV<T, DP, 4>><<<grid, 512, 0, s>>>(a);
    return hipGetLastError();
}

// Over the cache: 16 rows a wave whatever their number (32, which expand the
// codes half as often, hold one wave per SIMD at head 128 and two at 64: 2 x
// 4096 newest tokens of 32/8 heads of 128 took 501 us against 428, 64: 211 both),
// and the keys in shares where the rows are too few for the chip: 600 newest tokens of two
// sequences, 16/4 heads of 64 in fp16, window 2048, in 3 shares 38 us and 6 to
// join them, in two halves of a workgroup 49.
template <typename T, int DP>
hipError_t chunk(AttendArgs x, hipStream_t s) {
    const unsigned grid = tiles_of(x.a, 64, x.splits);
    attn_fwd_kernel<T, DP, 1, 4, 1, PagedKV<T, DP>><<<grid, 256, 0, s>>>(x);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_chunk(const AttendArgs &x, int dtype, hipStream_t s) {
    if (dtype == LSMX_BF16) return x.p.dim == 64 ? chunk<__bf16, 64>(x, s) : chunk<__bf16, 128>(x, s);
    return x.p.dim == 64 ? chunk<_Float16, 64>(x, s) : chunk<_Float16, 128>(x, s);
}

hipError_t launch_attn_fwd(const AttnArgs &a, int dtype, hipStream_t s) {
    if (dtype == LSMX_BF16) return a.dim <= 64 ? fwd<__bf16, 64>(a, s) : fwd<__bf16, 128>(a, s);
    return a.dim <= 64 ? fwd<_Float16, 64>(a, s) : fwd<_Float16, 128>(a, s);
}

}  // namespace lsmx
