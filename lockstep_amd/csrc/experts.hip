// The experts' products: rows in MXFP8 (E4M3 codes, one E8M0 scale for 32)
// times MXFP4 weights of the expert that each (token, slot) pair chose.
//
//   expert_gated    h_p = silu(x_t Wg^T) * (x_t Wu^T), in MXFP8
//   expert_combine  y_t = sum_j weight_tj (h_tj W^T)
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 4-bit weights and 8-bit rows as they
// lie in memory and applies both scales.  The weights are its A operand, so
// that a lane's four results are four rows of W for one pair.  Lane (i, g),
// g = lane / 16, supplies A's K 32g .. 32g+31 of row i, B's K 16g .. 16g+15
// and 64+16g .. of pair i, and block g's scales; its results are W's rows
// 4g .. 4g+3 for pair i.
//
// Pairs come sorted by expert (order, offsets); a workgroup finds the expert
// and the pairs of its tile from the offsets.  Nothing in order or offsets is
// trusted to be in range.
#include "lsmx_block.h"

namespace lsmx {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

__device__ v4f mfma_f4f8(v4i a, v8i b, v4f c, int cbsz, int blgp, int opsel_a, int scale_a, int opsel_b, int scale_b)
    __asm("llvm.amdgcn.mfma.scale.f32.16x16x128.f8f6f4.v4i32.v8i32");

namespace {

// A tile's pairs: order[start .. start + n), all of expert `expert`, or of no
// expert where that is `experts`.  n = 0: no tile.
struct Tile {
    int expert, start, n;
};

// Tile `slot` of all experts' pairs in tiles of `height`, then of the pairs of
// no expert.  Every wave computes it; experts <= 1024.
LSMX_DEV Tile find_tile(const int32_t *offsets, int experts, int pairs, int height, int slot) {
    const int lane = threadIdx.x & 63;
    const int per = (experts + 64) / 64;   // of experts + 1 entries
    // lane's entries: first .. first + per - 1
    const int first = lane * per;
    auto at = [&](int e) __attribute__((always_inline)) { return e > experts ? pairs : min(max(offsets[e], 0), pairs); };
    int mine = 0, lo = at(min(first, experts + 1));
    for (int i = 0; i < per; ++i) {
        const int hi = at(min(first + i + 1, experts + 1));
        if (first + i <= experts) mine += (max(hi - lo, 0) + height - 1) / height;
        lo = hi;
    }
    int inc = mine;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const int o = __shfl_up(inc, m, 64);
        if (lane >= m) inc += o;
    }
    const uint64_t past = __builtin_amdgcn_ballot_w64(inc > slot);
    if (!past) return Tile{0, 0, 0};
    const int owner = __builtin_ctzll(past);
    int left = slot - (__builtin_amdgcn_readlane(inc, owner) - __builtin_amdgcn_readlane(mine, owner));
    int e = owner * per;
    for (int i = 0; i < per; ++i, ++e) {
        const int lo2 = at(e), n = max(at(e + 1) - lo2, 0), tiles = (n + height - 1) / height;
        if (left < tiles) return Tile{e, lo2 + left * height, min(n - left * height, height)};
        left -= tiles;
    }
    return Tile{0, 0, 0};
}
// Slots that hold every tile, whatever the offsets.
int64_t tile_slots(int64_t pairs, int64_t experts, int64_t height) {
    return pairs / height + (experts + 1 < pairs ? experts + 1 : pairs);
}

LSMX_DEV float silu_times(float g, float u) { return g / (1.f + __expf(-g)) * u; }

// ------------------------------------------------------------ few rows
// A workgroup of KW waves: 64 rows of W (gated: 32 of the gate, the same 32 of
// up) for up to 16 NT pairs of one expert.  The waves split K, stream the
// weights from memory into registers and add their sums up in LDS.
template <bool GATED, int NT, int KW>
__global__ __launch_bounds__(64 * KW) void expert_stream_kernel(ExpertArgs a) {
    constexpr int C = 16 * NT;
    __shared__ __attribute__((aligned(16))) float sum[KW][64][C];
    __shared__ int pair_of[C];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), i16 = lane & 15, g = lane >> 4;
    const int blocks = (a.N + 63) / 64, nb = blockIdx.x % blocks;
    const Tile tile = find_tile(a.offsets, a.experts, a.pairs, C, blockIdx.x / blocks);
    if (tile.n == 0) return;
    if (t < C) {
        const uint32_t p = t < tile.n ? (uint32_t)a.order[tile.start + t] : 0xFFFFFFFFu;
        pair_of[t] = p < (uint32_t)a.pairs ? (int)p : -1;
    }
    __syncthreads();
    const int F = a.N / 2;
    if (tile.expert == a.experts) {   // pairs of no expert: rows of zeros
        if constexpr (GATED)
            for (int q = t; q < tile.n * 9; q += 64 * KW) {
                const int p = pair_of[q / 9], w = q % 9;
                if (p < 0) continue;
                if (w < 8)
                    *(uint32_t *)(a.h + (int64_t)p * F + nb * 32 + 4 * w) = 0;
                else
                    a.hs[(int64_t)p * (F / 32) + nb] = 127;
            }
        return;
    }
    const int kb = a.K / 32;
    // four tiles of 16 rows of W
    const uint8_t *wp[4], *sp[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int n0 = GATED ? nb * 32 + (r & 1) * 16 + (r >> 1) * F : nb * 64 + r * 16;
        const int64_t n = (int64_t)tile.expert * a.N + min(n0 + i16, a.N - 1);
        wp[r] = a.w + n * (a.K / 2) + 16 * g;
        sp[r] = a.ws + n * kb + g;
    }
    const uint8_t *xp[NT], *xsp[NT];
#pragma unroll
    for (int c = 0; c < NT; ++c) {
        const int p = max(pair_of[c * 16 + i16], 0);
        const int64_t row = GATED ? p / a.k : p;
        xp[c] = a.x + row * a.K + 16 * g;
        xsp[c] = a.xs + row * kb + g;
    }
    v4f acc[4][NT];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < NT; ++c) acc[r][c] = v4f{0.f, 0.f, 0.f, 0.f};
    const int steps = a.K / 128, s1 = steps * (wave + 1) / KW;
    for (int s = steps * wave / KW; s < s1; ++s) {
        v4i w[4];
        v8i x[NT];
        int ws[4], xs[NT];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            w[r] = *(const v4i *)(wp[r] + (int64_t)s * 64);
            ws[r] = sp[r][s * 4];
        }
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            const v4i lo = *(const v4i *)(xp[c] + (int64_t)s * 128), hi = *(const v4i *)(xp[c] + (int64_t)s * 128 + 64);
            x[c] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            xs[c] = xsp[c][s * 4];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < NT; ++c) acc[r][c] = mfma_f4f8(w[r], x[c], acc[r][c], 4, 0, 0, ws[r], 0, xs[c]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[wave][r * 16 + 4 * g + q][c * 16 + i16] = acc[r][c][q];
    __syncthreads();
    auto total = [&](int row, int col) __attribute__((always_inline)) {
        float v = sum[0][row][col];
#pragma unroll
        for (int w = 1; w < KW; ++w) v += sum[w][row][col];
        return v;
    };
    if constexpr (GATED) {
        // 8 threads a pair, 4 elements each
        for (int q = t; q < C * 8; q += 64 * KW) {
            const int c = q / 8, f = q % 8 * 4;
            float v[4];
            uint32_t am = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = silu_times(total(f + j, c), total(32 + f + j, c));
                am = max(am, f2u(v[j]) & 0x7FFFFFFFu);
            }
#pragma unroll
            for (int m = 1; m < 8; m *= 2) am = max(am, (uint32_t)__shfl_xor((int)am, m, 64));
            const uint32_t byte = mx8_byte(am);
            const float m = mx8_inverse(byte);
            const int p = pair_of[c];
            if (p >= 0) {
                *(uint32_t *)(a.h + (int64_t)p * F + nb * 32 + f) = e4m3_x4(v[0] * m, v[1] * m, v[2] * m, v[3] * m);
                if (f == 0) a.hs[(int64_t)p * (F / 32) + nb] = (uint8_t)byte;
            }
        }
    } else {
        for (int q = t; q < C * 64; q += 64 * KW) {
            const int c = q / 64, n = nb * 64 + q % 64, p = pair_of[c];
            if (p >= 0 && n < a.N) a.z[(int64_t)p * a.ldz + n] = total(q % 64, c);
        }
    }
}

// y_t = sum_j weight_tj z_tj over the pairs that have an expert, in the order of
// their slots.
template <int DT>
__global__ __launch_bounds__(256) void expert_join_kernel(ExpertArgs a) {
    typedef typename Elem<DT>::S S;
    const int64_t token = blockIdx.y + (int64_t)blockIdx.z * 65535;
    if (token >= a.tokens) return;
    const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (n >= a.N) return;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < a.k; ++j) {
        const int64_t p = token * a.k + j;
        if ((uint32_t)a.ids[p] >= (uint32_t)a.experts) continue;
        const float w = a.weights[p];
        const v4f z = *(const v4f *)(a.z + p * a.ldz + n);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += w * z[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < a.N) ((S *)a.y)[token * a.N + n + i] = Elem<DT>::store(v[i]);
}

template <bool GATED, int NT, int KW>
hipError_t stream(const ExpertArgs &a, hipStream_t s) {
    const int64_t slots = tile_slots(a.pairs, a.experts, 16 * NT);
    expert_stream_kernel<GATED, NT, KW><<<(unsigned)(slots * ((a.N + 63) / 64)), 64 * KW, 0, s>>>(a);
    return hipGetLastError();
}
template <bool GATED>
hipError_t products(const ExpertArgs &a, hipStream_t s) {
    const int64_t per = a.pairs / a.experts;
    return per <= 8 ? stream<GATED, 1, 8>(a, s) : stream<GATED, 4, 4>(a, s);
}

}  // namespace

hipError_t launch_expert_gated(const ExpertArgs &a, hipStream_t s) { return products<true>(a, s); }

hipError_t launch_expert_combine(const ExpertArgs &a, hipStream_t s) {
    hipError_t e = hipSuccess;
    if (a.pairs) e = products<false>(a, s);
    if (e != hipSuccess) return e;
    const dim3 grid((a.N + 1023) / 1024, (unsigned)(a.tokens < 65535 ? a.tokens : 65535), (unsigned)((a.tokens + 65534) / 65535));
    if (a.y_dtype == LSMX_F32)
        expert_join_kernel<LSMX_F32><<<grid, 256, 0, s>>>(a);
    else if (a.y_dtype == LSMX_BF16)
        expert_join_kernel<LSMX_BF16><<<grid, 256, 0, s>>>(a);
    else
        expert_join_kernel<LSMX_F16><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace lsmx
