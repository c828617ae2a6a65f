// A router's choice of experts, its gradient, and the pairs' order by expert.
//
//   s = softmax(l) or sigmoid(l),  c = s + b
//   a group of experts scores the sum of its two largest c; the top groups stay
//   i_1 .. i_k: the largest c of what stays, ties to the lowest index
//   w_j = scale s_ij / (renorm ? sum_j s_ij : 1)
//
// Choices are made in 64 bits: two scores may lie nearer to each other than
// 32 bits tell apart, and the choice is a whole number.
//
// Few rows are a matter of latency: 64 rows of 256 experts in 8 groups, sigmoid
// with a bias, 6.6 us.  Many are bound by the vector units, not by the logits'
// bytes: 30001 of those rows in 28 us, of which 6 are the bytes at a copy's rate;
// sorting a lane's 16 words, then a maximum over 16 lanes for each choice, is
// most of it.  Backward 30001 x 64 of bf16 5.4 us.
#include "lsmx_block.h"

namespace lsmx {

namespace {

// A lane's value from N lanes on, around its 16.
template <int N>
LSMX_DEV uint32_t ror16(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xF, 0xF, true);
}
template <int N>
LSMX_DEV double ror16(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)ror16<N>((uint32_t)(u >> 32)) << 32 | ror16<N>((uint32_t)u));
}
// max over 16 lanes, in all of them
LSMX_DEV uint32_t max16(uint32_t v) {
    v = max(v, ror16<1>(v));
    v = max(v, ror16<2>(v));
    v = max(v, ror16<4>(v));
    return max(v, ror16<8>(v));
}
LSMX_DEV float sum16(float v) {
    v += u2f(ror16<1>(f2u(v)));
    v += u2f(ror16<2>(f2u(v)));
    v += u2f(ror16<4>(f2u(v)));
    return v + u2f(ror16<8>(f2u(v)));
}
LSMX_DEV uint32_t lane_of(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }
LSMX_DEV double lane_of(double v, int l) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)lane_of((uint32_t)(u >> 32), l) << 32 | lane_of((uint32_t)u, l));
}
LSMX_DEV uint32_t wave_max(uint32_t v) {
    v = max16(v);
    return max(max(lane_of(v, 0), lane_of(v, 16)), max(lane_of(v, 32), lane_of(v, 48)));
}
LSMX_DEV double wave_sum(double v) {
    v += ror16<1>(v);
    v += ror16<2>(v);
    v += ror16<4>(v);
    v += ror16<8>(v);
    return lane_of(v, 0) + lane_of(v, 16) + (lane_of(v, 32) + lane_of(v, 48));
}
LSMX_DEV double wave_max(double v) {   // of numbers
    auto up = [](double p, double q) { return q > p ? q : p; };
    v = up(v, ror16<1>(v));
    v = up(v, ror16<2>(v));
    v = up(v, ror16<4>(v));
    v = up(v, ror16<8>(v));
    return up(up(lane_of(v, 0), lane_of(v, 16)), up(lane_of(v, 32), lane_of(v, 48)));
}
// order of the numbers as unsigned words: -0 is 0, a NaN above all; 0 is below all
LSMX_DEV uint64_t ordered(double f) {
    if (f != f) return ~0ull;
    const uint64_t u = __builtin_bit_cast(uint64_t, f + 0.0);
    return u ^ ((uint64_t)((int64_t)u >> 63) | 1ull << 63);
}

// The order in which values are chosen: a NaN before all, then the larger, of
// equal ones (-0 and 0 are equal) the lower index.
LSMX_DEV bool before(double a, int ia, double b, int ib) {
    const bool na = a != a, nb = b != b;
    if (na != nb) return na;
    if (!na && a != b) return a > b;
    return ia < ib;
}

template <int DT>
LSMX_DEV double logit(const RouteArgs &a, int64_t row, int e) {
    return (double)Elem<DT>::load(((const typename Elem<DT>::S *)a.logits)[row * a.ld + e]);
}

// Logits l and scores s of a row, NPL a lane (expert lane + 64 j); beyond the
// last: -inf and 0.  A row of nothing but -inf scores 0 throughout.
template <int DT, int NPL>
LSMX_DEV void scores(const RouteArgs &a, int64_t row, int lane, double (&l)[NPL], double (&s)[NPL]) {
#pragma unroll
    for (int j = 0; j < NPL; ++j) l[j] = lane + 64 * j < a.experts ? logit<DT>(a, row, lane + 64 * j) : -__builtin_inf();
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) s[j] = 1.0 / (1.0 + exp(-l[j]));
        return;
    }
    double m = -__builtin_inf(), t = 0.0;
#pragma unroll
    for (int j = 0; j < NPL; ++j) m = l[j] > m ? l[j] : m;
    m = wave_max(m);
#pragma unroll
    for (int j = 0; j < NPL; ++j) s[j] = l[j] == -__builtin_inf() ? 0.0 : exp(l[j] - m), t += s[j];
    t = wave_sum(t);
#pragma unroll
    for (int j = 0; j < NPL; ++j) s[j] = t == 0.0 ? 0.0 : s[j] / t;
}

// The row by a whole wave, in 64 bits throughout; row_of_c: `experts` doubles of
// LDS of its own, where there are groups.  Without a bias experts rank by
// their logits, the order of the scores.
template <int DT, int NPL>
LSMX_DEV void exact_row(const RouteArgs &a, int64_t row, int lane, double *row_of_c) {
    float *wo = a.weights + row * a.k;
    int32_t *io = a.ids + row * a.k;
    if (a.mask && !a.mask[row]) {
        if (lane < a.k) wo[lane] = 0.f, io[lane] = -1;
        return;
    }
    double l[NPL], s[NPL];
    uint64_t key[NPL];
    scores<DT, NPL>(a, row, lane, l, s);
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = lane + 64 * j;
        if (a.bias && e < a.experts) l[j] = s[j] + (double)a.bias[e];
        key[j] = e < a.experts ? ordered(l[j]) : 0;
    }
    if (a.top_groups < a.groups) {
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (key[j]) row_of_c[lane + 64 * j] = a.bias ? l[j] : s[j];
        __builtin_amdgcn_wave_barrier();
        const int size = a.experts / a.groups;
        // lane g scores group g (groups <= 64)
        double score = 0.0;
        if (lane < a.groups) {
            double u = row_of_c[lane * size], v = -__builtin_inf();
            for (int i = 1; i < size; ++i) {
                const double x = row_of_c[lane * size + i];
                if (before(x, 0, u, 1))
                    v = u, u = x;
                else if (before(x, 0, v, 1))
                    v = x;
            }
            score = size > 1 ? u + v : u;
        }
        // a group stays when fewer than top_groups are before it
        int ahead = 0;
        for (int g = 0; g < a.groups; ++g) ahead += g != lane && before(lane_of(score, g), g, score, lane);
        const uint64_t stay = __builtin_amdgcn_ballot_w64(lane < a.groups && ahead < a.top_groups);
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (!((stay >> (min(lane + 64 * j, a.experts - 1) / size)) & 1)) key[j] = 0;
        __builtin_amdgcn_wave_barrier();
    }
    float w = 0.f, total = 0.f;
    for (int j = 0; j < a.k; ++j) {
        // the first of this lane's, then of all lanes'
        uint64_t best = 0;
        int at = 0;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (key[i] > best) best = key[i], at = lane + 64 * i;
        const uint32_t hi = wave_max((uint32_t)(best >> 32)), lo = wave_max((uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
        const bool mine = best == ((uint64_t)hi << 32 | lo);
        const int first = 0xFFFF - (int)wave_max(mine ? 0xFFFFu - (uint32_t)at : 0u);
        float f = 0.f;
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            if (i == first >> 6) f = (float)s[i];
            if (lane + 64 * i == first) key[i] = 0;
        }
        f = u2f(lane_of(f2u(f), first & 63));
        if (lane == j) w = f, io[j] = first;
        total += f;
    }
    if (lane < a.k) wo[lane] = a.renorm ? (total == 0.f ? 0.f : a.scale * (w / total)) : a.scale * w;
}

template <int DT, int NPL>
__global__ __launch_bounds__(256) void route_fwd_kernel(RouteArgs a) {
    extern __shared__ double lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= a.rows) return;  // no barrier below: a wave works alone
    exact_row<DT, NPL>(a, row, lane, lds + wave * a.experts);
}

// ---------------------------------------------------------- 16 lanes a row
// Up to 256 experts and 16 choices: four rows a wave, V experts a lane (expert
// lane * v + j, v = ceil(experts / 16)).  Ranks are kept as words that order
// like the numbers, the index within the lane in the low bits; each lane sorts
// its own once, and a choice is then a maximum over 16 heads.
//
// Without a bias experts rank by their logits: 16-bit logits leave room for the
// whole index, and words never tie; fp32 ones lose 4 low bits, and tie where the
// others are equal.  With a bias ranks are fp32, and two of them may be wrong by
// both scores' errors (a sigmoid's 2.5e-7 each: exp, the sum, the reciprocal; a
// softmax's 2e-6 for both: the sum of up to 256 terms in 20 roundings), the
// additions' 2^-24 each and the 4 low bits, 15 * 2^-23 |c|: 2.2e-6 |c| and 6e-7
// or 2.2e-6.  A group's score adds two such errors.  Where two neighbours of the
// choice, or two groups, are too near to be told apart, the wave takes that row
// again in 64 bits.

// order of the numbers as unsigned words; 0 is below all
LSMX_DEV uint32_t ordered(float f) {
    const uint32_t u = f2u(f + 0.f);   // -0 as 0
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
LSMX_DEV float unordered(uint32_t u) { return u2f(u & 0x80000000u ? u ^ 0x80000000u : ~u); }

// descending, by merging (V a power of two)
template <int V>
LSMX_DEV void sort_down(uint32_t (&k)[V]) {
#pragma unroll
    for (int p = 1; p < V; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < V; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < V && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t x = max(k[i + j], k[i + j + q]), y = min(k[i + j], k[i + j + q]);
                        k[i + j] = x, k[i + j + q] = y;
                    }
}

// a lane's logits: v of them from expert lane * v on, -inf past the last
template <int DT, int V>
LSMX_DEV void lane_logits(const RouteArgs &a, int64_t row, int l16, int v, bool vec, float (&l)[V]) {
    typedef typename Elem<DT>::S S;
    const S *p = (const S *)a.logits + row * a.ld + l16 * v;
    constexpr int N = 16 / (int)sizeof(S) < V ? 16 / (int)sizeof(S) : V;
    typedef S W __attribute__((ext_vector_type(N)));
    if (vec) {
#pragma unroll
        for (int j = 0; j < V; j += N) {
            const W w = *(const W *)(p + j);
#pragma unroll
            for (int i = 0; i < N; ++i) l[j + i] = Elem<DT>::load(w[i]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) l[j] = Elem<DT>::load(p[min(j, a.experts - 1 - l16 * v)]);   // every lane loads something
#pragma unroll
        for (int j = 0; j < V; ++j) l[j] = j < v && l16 * v + j < a.experts ? l[j] : -__builtin_inff();
    }
}
// full vectors in every lane, aligned
template <int DT, int V>
LSMX_DEV bool whole_vectors(const RouteArgs &a, int v) {
    constexpr int N = (16 / (int)sizeof(typename Elem<DT>::S) < V ? 16 : V * (int)sizeof(typename Elem<DT>::S));
    return v == V && a.experts == 16 * V && (uintptr_t)a.logits % N == 0 && a.ld * (int)sizeof(typename Elem<DT>::S) % N == 0;
}

// within 2^-22 of 1
LSMX_DEV float sigmoid(float l) { return __builtin_amdgcn_rcpf(1.f + __expf(-l)); }

template <int DT, int V, int KM>   // k <= KM
__global__ __launch_bounds__(256) void route_fwd16_kernel(RouteArgs a) {
    constexpr int H = KM + 1 < V ? KM + 1 : V;   // of a lane's, those that can be chosen or be next
    extern __shared__ double lds[];   // a row of c for each wave, where there are groups
    __shared__ int chosen[16][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, r = threadIdx.x >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * 16 + wave * 4, row = row0 + (lane >> 4);
    if (row0 >= a.rows) return;   // no barrier below: a wave works alone
    const bool live = row < a.rows;
    const int64_t at = live ? row : a.rows - 1;
    const int v = (a.experts + 15) / 16;
    float l[V];
    lane_logits<DT, V>(a, at, l16, v, whole_vectors<DT, V>(a, v), l);
    const bool grouped = a.top_groups < a.groups, scored = a.bias != nullptr;
    // the row's largest logit, and whether 64 bits have to look at it
    uint32_t top = 0;
    bool odd = false;
#pragma unroll
    for (int j = 0; j < V; ++j) top = max(top, ordered(l[j])), odd |= !(l[j] < __builtin_inff());
    top = max16(top);
    const float m = unordered(top);
    // the sum of a softmax, where something needs it
    float inv = 1.f;
    const bool summed = !a.sigmoid && (scored || grouped || !a.renorm);
    if (summed) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) t += m == -__builtin_inff() ? 0.f : __expf(l[j] - m);
        t = sum16(t);
        inv = t > 0.f ? 1.f / t : 0.f;
    }
    auto score = [&](float x) __attribute__((always_inline)) {
        return a.sigmoid ? sigmoid(x) : x == -__builtin_inff() ? 0.f : __expf(x - m) * inv;
    };
    // ranks as words
    const bool whole = DT != LSMX_F32 && !scored;   // with the whole index
    const uint32_t low = whole ? (DT == LSMX_BF16 ? 0xFFFFu : 0x1FFFu) : 15u;
    uint32_t k[V];
    if (scored) {
        float c[V];
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] = a.bias[min(l16 * v + j, a.experts - 1)];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            c[j] += score(l[j]);
            odd |= !(c[j] < __builtin_inff());
            k[j] = ordered(c[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) k[j] = ordered(l[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int e = l16 * v + j;
        const uint32_t in = j < v && e < a.experts ? ~0u : 0u;
        k[j] = ((k[j] & ~low) | (low - (whole ? e : j))) & in;
    }
    sort_down<V>(k);
    bool near = false;
    const float off = a.sigmoid ? 6e-7f : 2.2e-6f;   // of two scores
    if (grouped) {
        // 16 / groups lanes a group: its two largest from their lanes' two
        uint32_t u = k[0], w = V > 1 ? k[1] : 0u;
        const int per = 16 / a.groups;
        auto merge = [&](uint32_t ou, uint32_t ow) __attribute__((always_inline)) {
            w = max(min(u, ou), max(w, ow));
            u = max(u, ou);
        };
        if (per > 1) merge(__shfl_xor((int)u, 1, 64), __shfl_xor((int)w, 1, 64));
        if (per > 2) merge(__shfl_xor((int)u, 2, 64), __shfl_xor((int)w, 2, 64));
        if (per > 4) merge(__shfl_xor((int)u, 4, 64), __shfl_xor((int)w, 4, 64));
        const float fu = unordered(u & ~low), fw = unordered(w & ~low);
        const bool two = a.experts > a.groups;   // else a group's one is its score
        // the group's score and how far it may be off
        float s, tol;
        if (scored) {
            s = fu + (two ? fw : 0.f);
            tol = 2.2e-6f * (__builtin_fabsf(fu) + __builtin_fabsf(two ? fw : 0.f)) + 2.f * off;
        } else {
            // a logit's lost bits change a softmax's score s by 15 * 2^-23 |l| s, a
            // sigmoid's by less than 0.23 of 15 * 2^-23
            const float su = score(fu), sw = two ? score(fw) : 0.f;
            s = su + sw;
            tol = 2.f * off + (a.sigmoid ? 1e-6f : 2e-6f * (su > 0.f ? su * __builtin_fabsf(fu) : 0.f) + 2e-6f * (sw > 0.f ? sw * __builtin_fabsf(fw) : 0.f));
        }
        const float lo = s - tol, hi = s + tol;
        // groups surely and perhaps ahead of this lane's
        int ahead = 0, perhaps = 0;
        auto look = [&](float olo, float ohi) __attribute__((always_inline)) {
            ahead += olo > hi;
            perhaps += !(ohi < lo);
        };
#define LOOK(n) look(u2f(ror16<n>(f2u(lo))), u2f(ror16<n>(f2u(hi))))
        LOOK(8);
        if (per <= 4) LOOK(4), LOOK(12);
        if (per <= 2) LOOK(2), LOOK(6), LOOK(10), LOOK(14);
        if (per <= 1) LOOK(1), LOOK(3), LOOK(5), LOOK(7), LOOK(9), LOOK(11), LOOK(13), LOOK(15);
#undef LOOK
        const bool out = ahead >= a.top_groups;
        near = !out && perhaps >= a.top_groups;
        if (out) {
#pragma unroll
            for (int j = 0; j < V; ++j) k[j] = 0;
        }
    }
    uint32_t last = 0;
    const int rounds = whole ? a.k : a.k + 1;   // one more to see whether the last choice is sure
    for (int j = 0; j < rounds; ++j) {
        const uint32_t best = max16(k[0]);
        const bool win = k[0] == best;
        if (win && j < a.k) chosen[r][j] = whole ? (int)(low - (best & low)) : l16 * v + (int)(low - (best & low));
        if (!whole && best != 0) {
            const uint32_t wins = (uint32_t)(__builtin_amdgcn_ballot_w64(win) >> (lane & 48)) & 0xFFFFu;
            near |= (wins & (wins - 1)) != 0;
            if (j > 0) {
                const float p = unordered(last & ~low), q = unordered(best & ~low);
                near |= scored ? !(p - q > 2.2e-6f * __builtin_fabsf(p) + off) : (last & ~low) == (best & ~low);
            }
        }
        last = best;
        const uint32_t up = win ? ~0u : 0u;
#pragma unroll
        for (int i = 0; i + 1 < H; ++i) k[i] = (k[i + 1] & up) | (k[i] & ~up);
        k[H - 1] &= ~up;
    }
    __builtin_amdgcn_wave_barrier();
    const bool masked = live && a.mask && !a.mask[row];
    const int id = l16 < a.k ? chosen[r][l16] : 0;
    // the chosen's scores, with the whole precision of exp
    auto exact = [&](float x) __attribute__((always_inline)) {
        return a.sigmoid ? 1.f / (1.f + expf(-x)) : x == -__builtin_inff() ? 0.f : expf(x - m) * inv;
    };
    float f = 0.f;
    if (l16 < a.k) f = exact(Elem<DT>::load(((const typename Elem<DT>::S *)a.logits)[at * a.ld + min((uint32_t)id, (uint32_t)(a.experts - 1))]));
    const float total = sum16(f);
    const float weight = a.renorm ? (total == 0.f ? 0.f : a.scale * (f / total)) : a.scale * f;
    uint64_t again = __builtin_amdgcn_ballot_w64(live && !masked && (odd || near));
    if (live && l16 < a.k && !(again >> (lane & 48) & 0xFFFF)) {
        a.weights[row * a.k + l16] = masked ? 0.f : weight;
        a.ids[row * a.k + l16] = masked ? -1 : id;
    }
    while (again) {   // a row at a time
        const int which = __builtin_ctzll(again) >> 4;
        exact_row<DT, (V + 3) / 4>(a, row0 + which, lane, lds + wave * a.experts);
        again &= ~(0xFFFFull << (16 * which));
    }
}

// The gradient with 16 lanes a row, in fp32.
template <int DT, int V>
__global__ __launch_bounds__(256) void route_bwd16_kernel(RouteArgs a) {
    typedef typename Elem<DT>::S S;
    __shared__ float g_of[16][16 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, r = threadIdx.x >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * 16 + wave * 4, row = row0 + (lane >> 4);
    if (row0 >= a.rows) return;   // no barrier below: a wave works alone
    const bool live = row < a.rows;
    const int64_t at = live ? row : a.rows - 1;
    const int v = (a.experts + 15) / 16;
    const bool vec = whole_vectors<DT, V>(a, v);
    const int id = l16 < a.k ? a.ids[at * a.k + l16] : -1;
    const float dw = l16 < a.k ? a.dw[at * a.k + l16] : 0.f;
    const bool there = (uint32_t)id < (uint32_t)a.experts;
    float l[V];
    lane_logits<DT, V>(a, at, l16, v, vec, l);
#pragma unroll
    for (int j = 0; j < V; ++j) g_of[r][l16 * V + j] = 0.f;
    float m = -__builtin_inff(), inv = 1.f;
    if (!a.sigmoid) {
        // a NaN stays one in the sum below
#pragma unroll
        for (int j = 0; j < V; ++j) m = fmaxf(m, l[j]);
        m = fmaxf(m, u2f(ror16<1>(f2u(m))));
        m = fmaxf(m, u2f(ror16<2>(f2u(m))));
        m = fmaxf(m, u2f(ror16<4>(f2u(m))));
        m = fmaxf(m, u2f(ror16<8>(f2u(m))));
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) l[j] = l[j] == -__builtin_inff() ? 0.f : expf(l[j] - m), t += l[j];
        t = sum16(t);
        inv = t == 0.f ? 0.f : 1.f / t;
    }
    auto score = [&](float x) __attribute__((always_inline)) {
        return a.sigmoid ? 1.f / (1.f + expf(-x)) : x == -__builtin_inff() ? 0.f : expf(x - m) * inv;
    };
    const float own = there ? score(Elem<DT>::load(((const S *)a.logits)[at * a.ld + id])) : 0.f;
    float g = a.scale * dw;
    if (a.renorm) {
        const float total = sum16(own), da = sum16(dw * own);
        g = total == 0.f ? 0.f : a.scale * (dw - da / total) / total;
    }
    if (!there) g = 0.f;
    const float mean = sum16(g * own);
    __builtin_amdgcn_wave_barrier();
    if (there) g_of[r][id / v * V + id % v] = g;
    __builtin_amdgcn_wave_barrier();
    const bool any = (__builtin_amdgcn_ballot_w64(there) >> (lane & 48)) & 0xFFFF;   // a masked row has no gradient
    float d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float x = g_of[r][l16 * V + j];
        if (a.sigmoid) {
            const float s = score(l[j]);
            d[j] = x == 0.f ? 0.f : x * s * (1.f - s);
        } else {
            d[j] = l[j] * inv * (x - mean);
        }
        if (!any) d[j] = 0.f;
    }
    if (!live) return;
    S *out = (S *)a.dlogits + row * a.experts + l16 * v;
    constexpr int N = 16 / (int)sizeof(S) < V ? 16 / (int)sizeof(S) : V;
    typedef S W __attribute__((ext_vector_type(N)));
    if (vec && (uintptr_t)a.dlogits % 16 == 0) {
#pragma unroll
        for (int j = 0; j < V; j += N) {
            W w;
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = Elem<DT>::store(d[j + i]);
            *(W *)(out + j) = w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < v && l16 * v + j < a.experts) out[j] = Elem<DT>::store(d[j]);
    }
}

template <int DT, int NPL>
__global__ __launch_bounds__(256) void route_bwd_kernel(RouteArgs a) {
    typedef typename Elem<DT>::S S;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= a.rows) return;
    S *out = (S *)a.dlogits + row * a.experts;
    double l[NPL], s[NPL], d[NPL];
    scores<DT, NPL>(a, row, lane, l, s);
    const int id = lane < a.k ? a.ids[row * a.k + lane] : -1;
    const double dw = lane < a.k ? (double)a.dw[row * a.k + lane] : 0.0;
    // a lane's chosen score, then the sums over the chosen
    double own = 0.0;
    for (int j = 0; j < a.k; ++j) {
        const int e = __builtin_amdgcn_readlane(id, j);
        if (e < 0 || e >= a.experts) continue;
        double v = 0.0;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (i == e / 64) v = s[i];
        v = lane_of(v, e & 63);
        if (lane == j) own = v;
    }
    const double total = wave_sum(own), da = wave_sum(dw * own);
    double g = a.scale * dw;   // gradient of a lane's chosen score
    if (a.renorm) g = total == 0.0 ? 0.0 : a.scale * (dw - da / total) / total;
    if (id < 0) g = 0.0;
    const double mean = wave_sum(g * own);
#pragma unroll
    for (int i = 0; i < NPL; ++i) d[i] = 0.0;
    for (int j = 0; j < a.k; ++j) {
        const int e = __builtin_amdgcn_readlane(id, j);
        const double v = lane_of(g, j);
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (e == lane + 64 * i) d[i] = v;
    }
    const bool any = __builtin_amdgcn_ballot_w64(id >= 0) != 0;   // a masked row has no gradient
#pragma unroll
    for (int i = 0; i < NPL; ++i)
        if (lane + 64 * i < a.experts) {
            const double v = a.sigmoid ? (d[i] == 0.0 ? 0.0 : d[i] * s[i] * (1.0 - s[i])) : s[i] * (d[i] - mean);
            out[lane + 64 * i] = Elem<DT>::store(any ? (float)v : 0.f);
        }
}

template <int DT, int V>
void fwd16(const RouteArgs &a, unsigned grid, size_t lds, hipStream_t s) {
    if (a.k <= 8)
        route_fwd16_kernel<DT, V, 8><<<grid, 256, lds, s>>>(a);
    else
        route_fwd16_kernel<DT, V, 16><<<grid, 256, lds, s>>>(a);
}

// What 16 lanes a row take: their experts in registers, the groups as whole
// lanes.  One row that 64 bits have to look at makes the call as long as the
// other kernel and more: with a bias or groups, a few rows rarely have one, many
// have the time; between them the other kernel is quicker (us, 256 experts,
// sigmoid with a bias: 64 rows 6.2 against 6.3, 1024 10.2 against 6.7, 4096 10.4
// against 9.5, 8192 12.6 against 14.5; in 8 groups 6.6 against 9.6, 12.7 against
// 9.5, 13.0 against 13.1, 16.0 against 21.5).
bool in16(const RouteArgs &a) {
    const bool grouped = a.top_groups < a.groups;
    return a.experts <= 256 && a.k <= 16 && (!grouped || (a.experts % 16 == 0 && 16 % a.groups == 0)) &&
           ((!a.bias && !grouped) || a.rows <= 128 || a.rows > 4096);
}

template <int DT>
hipError_t fwd_of(const RouteArgs &a, hipStream_t s) {
    const size_t lds = a.top_groups < a.groups ? (size_t)a.experts * 4 * sizeof(double) : 0;
    if (in16(a)) {
        const unsigned grid = (unsigned)((a.rows + 15) / 16);
        if (a.experts <= 16)
            fwd16<DT, 1>(a, grid, lds, s);
        else if (a.experts <= 32)
            fwd16<DT, 2>(a, grid, lds, s);
        else if (a.experts <= 64)
            fwd16<DT, 4>(a, grid, lds, s);
        else if (a.experts <= 128)
            fwd16<DT, 8>(a, grid, lds, s);
        else
            fwd16<DT, 16>(a, grid, lds, s);
        return hipGetLastError();
    }
    const unsigned grid = (unsigned)((a.rows + 3) / 4);
    if (a.experts <= 64)
        route_fwd_kernel<DT, 1><<<grid, 256, lds, s>>>(a);
    else if (a.experts <= 128)
        route_fwd_kernel<DT, 2><<<grid, 256, lds, s>>>(a);
    else if (a.experts <= 256)
        route_fwd_kernel<DT, 4><<<grid, 256, lds, s>>>(a);
    else if (a.experts <= 512)
        route_fwd_kernel<DT, 8><<<grid, 256, lds, s>>>(a);
    else
        route_fwd_kernel<DT, 16><<<grid, 256, lds, s>>>(a);
    return hipGetLastError();
}
template <int DT>
hipError_t bwd_of(const RouteArgs &a, hipStream_t s) {
    if (a.experts <= 256 && a.k <= 16) {
        const unsigned grid = (unsigned)((a.rows + 15) / 16);
        if (a.experts <= 16)
            route_bwd16_kernel<DT, 1><<<grid, 256, 0, s>>>(a);
        else if (a.experts <= 32)
            route_bwd16_kernel<DT, 2><<<grid, 256, 0, s>>>(a);
        else if (a.experts <= 64)
            route_bwd16_kernel<DT, 4><<<grid, 256, 0, s>>>(a);
        else if (a.experts <= 128)
            route_bwd16_kernel<DT, 8><<<grid, 256, 0, s>>>(a);
        else
            route_bwd16_kernel<DT, 16><<<grid, 256, 0, s>>>(a);
        return hipGetLastError();
    }
    const unsigned grid = (unsigned)((a.rows + 3) / 4);
    if (a.experts <= 64)
        route_bwd_kernel<DT, 1><<<grid, 256, 0, s>>>(a);
    else if (a.experts <= 128)
        route_bwd_kernel<DT, 2><<<grid, 256, 0, s>>>(a);
    else if (a.experts <= 256)
        route_bwd_kernel<DT, 4><<<grid, 256, 0, s>>>(a);
    else if (a.experts <= 512)
        route_bwd_kernel<DT, 8><<<grid, 256, 0, s>>>(a);
    else
        route_bwd_kernel<DT, 16><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

// ---------------------------------------------------------------- dispatch
// The pairs sorted by expert, stable: a counting sort.  A workgroup takes ROUNDS
// times 1024 pairs, each of its waves consecutive ones in rounds of 64; lanes of
// one expert find their rank from the ballots of its bits.  Ids outside the
// experts count as expert `experts`, behind the others.

// One round of a wave: each lane's rank among the wave's pairs of its expert so
// far, the counts brought up to date.
LSMX_DEV int round_rank(int e, int bits, uint16_t *hist, bool live) {
    uint64_t same = __builtin_amdgcn_ballot_w64(live);
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __builtin_amdgcn_ballot_w64((e >> b) & 1);
        same &= (e >> b) & 1 ? set : ~set;
    }
    const int lane = threadIdx.x & 63;
    const int below = __builtin_popcountll(same & ((1ull << lane) - 1));
    int rank = 0;
    if (live) rank = hist[e] + below;
    __builtin_amdgcn_wave_barrier();
    if (live && below == 0) hist[e] = (uint16_t)(rank + __builtin_popcountll(same));
    __builtin_amdgcn_wave_barrier();
    return rank;
}
// of pair p, or of the last one (loads without conditions go out together)
LSMX_DEV int expert_of(const int32_t *ids, int p, int pairs, int experts) {
    return (int)min((uint32_t)ids[min(p, pairs - 1)], (uint32_t)experts);
}

// counts[block][expert]: the pairs of each workgroup
template <int ROUNDS>
__global__ __launch_bounds__(1024) void dispatch_count_kernel(const int32_t *ids, int pairs, int experts, int32_t *counts) {
    extern __shared__ int hist1[];
    const int first = blockIdx.x * 1024 * ROUNDS + threadIdx.x;
    int e[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) e[r] = expert_of(ids, first + 1024 * r, pairs, experts);
    for (int i = threadIdx.x; i <= experts; i += 1024) hist1[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (first + 1024 * r < pairs) atomicAdd(&hist1[e[r]], 1);
    __syncthreads();
    for (int i = threadIdx.x; i <= experts; i += 1024) counts[(int64_t)blockIdx.x * (experts + 1) + i] = hist1[i];
}

// order and offsets.  counts null: one workgroup, which counts for itself.
template <int ROUNDS>
__global__ __launch_bounds__(1024) void dispatch_kernel(const int32_t *ids, int pairs, int experts, int bits,
                                                        const int32_t *counts, int32_t *order, int32_t *offsets) {
    extern __shared__ int lds_i[];   // bases [experts + 1], totals [experts + 1], counts [waves][experts + 1]
    const int threads = blockDim.x, waves = threads / 64;
    const int n = experts + 1;
    int *base = lds_i, *scan = lds_i + n;
    uint16_t *hists = (uint16_t *)(lds_i + 2 * n);   // at most 1024 ROUNDS
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint16_t *hist = hists + wave * n;
    const int first = blockIdx.x * 1024 * ROUNDS + wave * (64 * ROUNDS) + lane;
    int e[ROUNDS], rank[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) e[r] = pairs ? expert_of(ids, first + 64 * r, pairs, experts) : 0;
    for (int i = t; i < waves * n; i += threads) hists[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) rank[r] = round_rank(e[r], bits, hist, first + 64 * r < pairs);
    __syncthreads();
    // expert x: pairs of earlier workgroups, of all, and the waves' counts turned
    // into where each begins
    for (int x = t; x < n; x += threads) {
        int run = 0;
        for (int w = 0; w < waves; ++w) {
            const int c = hists[w * n + x];
            hists[w * n + x] = (uint16_t)run;
            run += c;
        }
        int before = 0, all = run;
        if (counts) {
            all = 0;
            for (int b = 0; b < (int)gridDim.x; b += 8) {   // eight loads at a time
                int c[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) c[i] = counts[(int64_t)min(b + i, (int)gridDim.x - 1) * n + x];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    before += b + i < (int)blockIdx.x ? c[i] : 0;
                    all += b + i < (int)gridDim.x ? c[i] : 0;
                }
            }
        }
        base[x] = before;
        scan[x] = all;
    }
    __syncthreads();
    // exclusive scan of the totals, by the first wave
    if (wave == 0) {
        int carry = 0;
        for (int x0 = 0; x0 < n; x0 += 64) {
            const int x = x0 + lane;
            const int v = x < n ? scan[x] : 0;
            const int inc = scan64(v);
            if (x < n) scan[x] = carry + inc - v;
            carry += __builtin_amdgcn_readlane(inc, 63);
        }
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int x = t; x < n; x += threads) offsets[x] = scan[x];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int p = first + 64 * r;
        if (p < pairs) order[scan[e[r]] + base[e[r]] + hist[e[r]] + rank[r]] = p;
    }
}

}  // namespace

// `launch` over all rows: a launch has fewer than 2^32 threads.
template <typename L>
static hipError_t in_parts(const RouteArgs &a0, L launch) {
    RouteArgs a = a0;
    const int64_t most = 1 << 22, es = a.dtype == LSMX_F32 ? 4 : 2;
    for (int64_t at = 0; at < a0.rows; at += most) {
        a.rows = a0.rows - at < most ? a0.rows - at : most;
        a.logits = (const uint8_t *)a0.logits + at * a.ld * es;
        a.mask = a0.mask ? a0.mask + at : nullptr;
        a.weights = a0.weights ? a0.weights + at * a.k : nullptr;
        a.ids = a0.ids + at * a.k;
        a.dw = a0.dw ? a0.dw + at * a.k : nullptr;
        a.dlogits = a0.dlogits ? (uint8_t *)a0.dlogits + at * a.experts * es : nullptr;
        const hipError_t e = launch(a);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
hipError_t launch_route_fwd(const RouteArgs &a0, hipStream_t s) {
    return in_parts(a0, [s](const RouteArgs &a) {
        return a.dtype == LSMX_F32 ? fwd_of<LSMX_F32>(a, s) : a.dtype == LSMX_BF16 ? fwd_of<LSMX_BF16>(a, s) : fwd_of<LSMX_F16>(a, s);
    });
}
hipError_t launch_route_bwd(const RouteArgs &a0, hipStream_t s) {
    return in_parts(a0, [s](const RouteArgs &a) {
        return a.dtype == LSMX_F32 ? bwd_of<LSMX_F32>(a, s) : a.dtype == LSMX_BF16 ? bwd_of<LSMX_BF16>(a, s) : bwd_of<LSMX_F16>(a, s);
    });
}

// Rounds of a workgroup of 16 waves, 1024 pairs each.  One workgroup needs no
// counting before it: 2000 pairs of 32 experts in two rounds 3.7 us, with it 5.2.
// More workgroups have fewer rounds but more counts to add up: 4096 pairs in four
// rounds 5.4, in four workgroups 5.2 (128 experts 6.7 and 5.6); 32768 in eight
// workgroups of four rounds 8.2, in 32 of one 6.8; 65536 9.1 and 8.3; 2^21 in 512
// workgroups 37.
static int dispatch_rounds(int64_t pairs) { return pairs <= 1024 ? 1 : pairs <= 2048 ? 2 : pairs <= 65536 ? 1 : 4; }

int64_t dispatch_workspace(int64_t pairs, int experts) {
    const int64_t each = 1024 * dispatch_rounds(pairs), blocks = (pairs + each - 1) / each;
    return blocks > 1 ? blocks * (experts + 1) * 4 : 0;
}

namespace {
template <int ROUNDS>
hipError_t dispatch(const int32_t *ids, int pairs, int experts, int32_t *order, int32_t *offsets, int32_t *ws, hipStream_t s) {
    const int blocks = pairs ? (pairs + 1024 * ROUNDS - 1) / (1024 * ROUNDS) : 1;
    if (blocks > 1) {
        dispatch_count_kernel<ROUNDS><<<blocks, 1024, (experts + 1) * 4, s>>>(ids, pairs, experts, ws);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    int bits = 1;
    while ((1 << bits) <= experts) ++bits;
    // up to 1024 pairs: a round for each wave, as many waves as it takes
    const int waves = pairs <= 1024 ? (pairs + 63) / 64 + (pairs == 0) : 16;
    dispatch_kernel<ROUNDS><<<blocks, 64 * waves, (size_t)(experts + 1) * (8 + 2 * waves), s>>>(ids, pairs, experts, bits, blocks > 1 ? ws : nullptr,
                                                                                         order, offsets);
    return hipGetLastError();
}
}  // namespace

hipError_t launch_dispatch(const int32_t *ids, int pairs, int experts, int32_t *order, int32_t *offsets, int32_t *ws,
                           hipStream_t s) {
    switch (dispatch_rounds(pairs)) {
        case 1: return dispatch<1>(ids, pairs, experts, order, offsets, ws, s);
        case 2: return dispatch<2>(ids, pairs, experts, order, offsets, ws, s);
        default: return dispatch<4>(ids, pairs, experts, order, offsets, ws, s);
    }
}

}  // namespace lsmx
