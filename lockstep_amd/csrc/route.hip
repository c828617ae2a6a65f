// A router's choice of experts, its gradient, and the pairs' order by expert.
//
//   s = softmax(l) or sigmoid(l),  c = s + b
//   a group of experts scores the sum of its two largest c; the top groups stay
//   i_1 .. i_k: the largest c of what stays, ties to the lowest index
//   w_j = scale s_ij / (renorm ? sum_j s_ij : 1)
//
// Choices are made in 64 bits: two scores may lie nearer to each other than
// 32 bits tell apart, and the choice is a whole number.
#include "lsmx_block.h"

namespace lsmx {

namespace {

LSMX_DEV double shfl_d(double v, int m) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)u, m, 64), hi = (uint32_t)__shfl_xor((int)(uint32_t)(u >> 32), m, 64);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
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

// Scores of a row, NPL a lane (expert lane + 64 j); beyond the last: -inf in
// `l` and 0 in `s`.  A row of nothing but -inf scores 0 throughout.
template <int DT, int NPL>
LSMX_DEV void scores(const RouteArgs &a, int64_t row, int lane, double (&s)[NPL]) {
    double l[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) l[j] = lane + 64 * j < a.experts ? logit<DT>(a, row, lane + 64 * j) : -__builtin_inf();
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) s[j] = 1.0 / (1.0 + exp(-l[j]));
        return;
    }
    double m = -__builtin_inf();
    bool nan = false;
#pragma unroll
    for (int j = 0; j < NPL; ++j) m = l[j] > m ? l[j] : m, nan |= l[j] != l[j];
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
        const double o = shfl_d(m, x);
        m = o > m ? o : m;
    }
    double t = 0.0;
#pragma unroll
    for (int j = 0; j < NPL; ++j) s[j] = m == -__builtin_inf() && !nan ? 0.0 : exp(l[j] - m), t += s[j];
#pragma unroll
    for (int x = 1; x < 64; x *= 2) t += shfl_d(t, x);
#pragma unroll
    for (int j = 0; j < NPL; ++j) s[j] = t == 0.0 ? 0.0 : s[j] / t;
}

template <int DT, int NPL>
__global__ __launch_bounds__(256) void route_fwd_kernel(RouteArgs a) {
    extern __shared__ double lds[];  // a wave's row of c, where there are groups
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= a.rows) return;  // no barrier below: a wave works alone
    float *wo = a.weights + row * a.k;
    int32_t *io = a.ids + row * a.k;
    if (a.mask && !a.mask[row]) {
        if (lane < a.k) wo[lane] = 0.f, io[lane] = -1;
        return;
    }
    double s[NPL], c[NPL];
    bool live[NPL];
    scores<DT, NPL>(a, row, lane, s);
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = lane + 64 * j;
        live[j] = e < a.experts;
        c[j] = a.bias && live[j] ? s[j] + (double)a.bias[e] : s[j];
    }
    if (a.top_groups < a.groups) {
        double *mine = lds + wave * a.experts;
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (live[j]) mine[lane + 64 * j] = c[j];
        __builtin_amdgcn_wave_barrier();
        const int size = a.experts / a.groups;
        // lane g scores group g (groups <= 64)
        double score = 0.0;
        if (lane < a.groups) {
            double u = mine[lane * size], v = -__builtin_inf();
            for (int i = 1; i < size; ++i) {
                const double x = mine[lane * size + i];
                if (before(x, 0, u, 1))
                    v = u, u = x;
                else if (before(x, 0, v, 1))
                    v = x;
            }
            score = size > 1 ? u + v : u;
        }
        // a group stays when fewer than top_groups are before it
        int ahead = 0;
        for (int g = 0; g < a.groups; ++g) {
            const uint64_t u = __builtin_bit_cast(uint64_t, score);
            const double o = __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(u >> 32), g) << 32 |
                                                            (uint32_t)__builtin_amdgcn_readlane((uint32_t)u, g));
            ahead += g != lane && before(o, g, score, lane);
        }
        const uint64_t stay = __builtin_amdgcn_ballot_w64(lane < a.groups && ahead < a.top_groups);
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (live[j]) live[j] = (stay >> ((lane + 64 * j) / size)) & 1;
    }
    float w = 0.f, total = 0.f;
    for (int j = 0; j < a.k; ++j) {
        // the first of this lane's, then of all lanes'
        double best = -__builtin_inf(), sc = 0.0;
        int at = 0x7FFFFFFF;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (live[i] && (at == 0x7FFFFFFF || before(c[i], lane + 64 * i, best, at))) best = c[i], at = lane + 64 * i, sc = s[i];
        int first = at;
        double fb = best;
#pragma unroll
        for (int x = 1; x < 64; x *= 2) {
            const double ob = shfl_d(fb, x);
            const int oa = __shfl_xor(first, x, 64);
            if (oa != 0x7FFFFFFF && (first == 0x7FFFFFFF || before(ob, oa, fb, first))) fb = ob, first = oa;
        }
        const int from = first & 63;
        const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, (float)sc), __builtin_amdgcn_readfirstlane(from)));
        if (lane == j) w = f, io[j] = first;
        total += f;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (lane + 64 * i == first) live[i] = false;
    }
    if (lane < a.k) wo[lane] = a.renorm ? (total == 0.f ? 0.f : a.scale * (w / total)) : a.scale * w;
}

template <int DT, int NPL>
__global__ __launch_bounds__(256) void route_bwd_kernel(RouteArgs a) {
    typedef typename Elem<DT>::S S;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= a.rows) return;
    S *out = (S *)a.dlogits + row * a.experts;
    double s[NPL], d[NPL];
    scores<DT, NPL>(a, row, lane, s);
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
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        v = __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(u >> 32), e & 63) << 32 |
                                           (uint32_t)__builtin_amdgcn_readlane((uint32_t)u, e & 63));
        if (lane == j) own = v;
    }
    double total = own, da = dw * own;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) total += shfl_d(total, x), da += shfl_d(da, x);
    double g = a.scale * dw;   // gradient of a lane's chosen score
    if (a.renorm) g = total == 0.0 ? 0.0 : a.scale * (dw - da / total) / total;
    if (id < 0) g = 0.0;
    double mean = g * own;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) mean += shfl_d(mean, x);
#pragma unroll
    for (int i = 0; i < NPL; ++i) d[i] = 0.0;
    for (int j = 0; j < a.k; ++j) {
        const int e = __builtin_amdgcn_readlane(id, j);
        const uint64_t u = __builtin_bit_cast(uint64_t, g);
        const double v = __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(u >> 32), j) << 32 |
                                                        (uint32_t)__builtin_amdgcn_readlane((uint32_t)u, j));
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

template <int DT>
hipError_t fwd_of(const RouteArgs &a, hipStream_t s) {
    const unsigned grid = (unsigned)((a.rows + 3) / 4);
    const size_t lds = a.top_groups < a.groups ? (size_t)a.experts * 4 * sizeof(double) : 0;
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
// The pairs sorted by expert, stable: a counting sort.  A workgroup takes 4096
// pairs, each of its waves 256 consecutive ones in rounds of 64; lanes of one
// expert find their rank from the ballots of its bits.  Ids outside the
// experts count as expert `experts`, behind the others.
constexpr int kDispWaves = 16, kDispPairs = 4096;

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
LSMX_DEV int expert_of(const int32_t *ids, int p, int experts) {
    const uint32_t e = (uint32_t)ids[p];
    return e < (uint32_t)experts ? (int)e : experts;
}

// counts[block][expert]: the pairs of each workgroup
__global__ __launch_bounds__(1024) void dispatch_count_kernel(const int32_t *ids, int pairs, int experts, int32_t *counts) {
    extern __shared__ int hist1[];
    for (int i = threadIdx.x; i <= experts; i += 1024) hist1[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < kDispPairs; i += 1024) {
        const int p = blockIdx.x * kDispPairs + i;
        if (p < pairs) atomicAdd(&hist1[expert_of(ids, p, experts)], 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i <= experts; i += 1024) counts[(int64_t)blockIdx.x * (experts + 1) + i] = hist1[i];
}

// order and offsets.  counts null: one workgroup, which counts for itself.
__global__ __launch_bounds__(1024) void dispatch_kernel(const int32_t *ids, int pairs, int experts, int bits,
                                                        const int32_t *counts, int32_t *order, int32_t *offsets) {
    extern __shared__ int lds_i[];   // bases [experts + 1], totals [experts + 1], counts [waves][experts + 1]
    const int n = experts + 1;
    int *base = lds_i, *scan = lds_i + n;
    uint16_t *hists = (uint16_t *)(lds_i + 2 * n);   // at most kDispPairs
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    for (int i = t; i < kDispWaves * n; i += 1024) hists[i] = 0;
    __syncthreads();
    uint16_t *hist = hists + wave * n;
    int e[kDispPairs / 1024], rank[kDispPairs / 1024];
#pragma unroll
    for (int r = 0; r < kDispPairs / 1024; ++r) {
        const int p = blockIdx.x * kDispPairs + wave * (kDispPairs / kDispWaves) + r * 64 + lane;
        const bool live = p < pairs;
        e[r] = live ? expert_of(ids, p, experts) : 0;
        rank[r] = round_rank(e[r], bits, hist, live);
    }
    __syncthreads();
    // expert x: pairs of earlier workgroups, of all, and the waves' counts turned
    // into where each begins
    for (int x = t; x < n; x += 1024) {
        int run = 0;
        for (int w = 0; w < kDispWaves; ++w) {
            const int c = hists[w * n + x];
            hists[w * n + x] = (uint16_t)run;
            run += c;
        }
        int before = 0, all = run;
        if (counts) {
            all = 0;
            for (int b = 0; b < (int)gridDim.x; ++b) {
                const int c = counts[(int64_t)b * n + x];
                before += b < (int)blockIdx.x ? c : 0;
                all += c;
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
            int inc = v;
#pragma unroll
            for (int m = 1; m < 64; m *= 2) {
                const int o = __shfl_up(inc, m, 64);
                if (lane >= m) inc += o;
            }
            if (x < n) scan[x] = carry + inc - v;
            carry += __shfl(inc, 63, 64);
        }
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int x = t; x < n; x += 1024) offsets[x] = scan[x];
#pragma unroll
    for (int r = 0; r < kDispPairs / 1024; ++r) {
        const int p = blockIdx.x * kDispPairs + wave * (kDispPairs / kDispWaves) + r * 64 + lane;
        if (p < pairs) order[scan[e[r]] + base[e[r]] + hist[e[r]] + rank[r]] = p;
    }
}

}  // namespace

hipError_t launch_route_fwd(const RouteArgs &a, hipStream_t s) {
    return a.dtype == LSMX_F32 ? fwd_of<LSMX_F32>(a, s) : a.dtype == LSMX_BF16 ? fwd_of<LSMX_BF16>(a, s) : fwd_of<LSMX_F16>(a, s);
}
hipError_t launch_route_bwd(const RouteArgs &a, hipStream_t s) {
    return a.dtype == LSMX_F32 ? bwd_of<LSMX_F32>(a, s) : a.dtype == LSMX_BF16 ? bwd_of<LSMX_BF16>(a, s) : bwd_of<LSMX_F16>(a, s);
}

int64_t dispatch_workspace(int64_t pairs, int experts) {
    const int64_t blocks = (pairs + kDispPairs - 1) / kDispPairs;
    return blocks > 1 ? blocks * (experts + 1) * 4 : 0;
}
hipError_t launch_dispatch(const int32_t *ids, int pairs, int experts, int32_t *order, int32_t *offsets, int32_t *ws,
                           hipStream_t s) {
    const int blocks = pairs ? (pairs + kDispPairs - 1) / kDispPairs : 1;
    int bits = 1;
    while ((1 << bits) <= experts) ++bits;
    if (blocks > 1) {
        dispatch_count_kernel<<<blocks, 1024, (experts + 1) * 4, s>>>(ids, pairs, experts, ws);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    const size_t lds = (size_t)(experts + 1) * (8 + 2 * kDispWaves);
    dispatch_kernel<<<blocks, 1024, lds, s>>>(ids, pairs, experts, bits, blocks > 1 ? ws : nullptr, order, offsets);
    return hipGetLastError();
}

}  // namespace lsmx
