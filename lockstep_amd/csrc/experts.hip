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
// 4g .. 4g+3 for pair i (checked on the device against the products).
//
// The instruction adds eight products at a time, keeping 13 bits below the
// largest exponent among them; beyond those eight its sums are fp32.  E4M3 spans
// more than that: rows with both large and small codes lose 4e-6 of a result
// (rms, normal values).  The forms that wait for memory take each row's codes of
// 2 and more and those below in two instructions, which is exact; the forms for
// many rows, bound by the matrix cores, do not (twice the instructions).
//
// What bounds them.  Few rows: an expert's weights are read once, F N 17/32
// bytes each, at the rate of a large copy (4.9 TB/s): 64 tokens that choose 8 of
// 128 experts, K = 4096, F = 1024, read nearly all of 571 MB in 110 us.  Many
// rows: the matrix cores, which alone, from registers, run these types at 3.6
// PF/s; 8192 tokens of 4 of 32 experts, K = 4096, F = 2048 take 460 us gated
// (2.4 PF/s; codes and weights through LDS keep them busy half of the time, the
// gate and its rounding are a tenth of a tile), 362 us combined (K = 2048, N =
// 4096; the products 250 us, a pair's rows written and read 110).
//
// Pairs come sorted by expert (order, offsets); a workgroup finds the expert
// and the pairs of its tile from the offsets.  Nothing in order or offsets is
// trusted to be in range.
#include "lsmx_block.h"
#include "lsmx_dma.h"
#include "lsmx_internal.h"

namespace lsmx {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

__device__ v4f mfma_f4f8(v4i a, v8i b, v4f c, int cbsz, int blgp, int opsel_a, int scale_a, int opsel_b, int scale_b)
    __asm("llvm.amdgcn.mfma.scale.f32.16x16x128.f8f6f4.v4i32.v8i32");

namespace {

// The codes of magnitude 2 and more (bit 6 of a byte), the others 0.
LSMX_DEV v8i large_codes(v8i x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = (uint32_t)x[i] & 0x40404040u;
        x[i] &= (int)((b << 2) - (b >> 6));
    }
    return x;
}

// Maximum over the four lanes of a pair (lane, lane ^ 16, ..).
LSMX_DEV uint32_t max4(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(b[0], b[1]);
}
// Lane g has pieces 4g .. of two tiles of 16 rows, p and q; it gets pieces 2g and
// 2g + 1 of the 32 rows, so that its store is twice as wide and a pair's four
// are neighbours.
LSMX_DEV void neighbours(uint32_t &p, uint32_t &q) {
    const auto a = __builtin_amdgcn_permlane32_swap(p, q, false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(a[0], a[1], false, false);
    p = b[0], q = b[1];
}

// ---------------------------------------------------------------- the tiles
// What a workgroup does: block `block` of W's rows for the pairs
// order[start .. start + n), all of expert `expert`, or of no expert where that
// is `experts`.  n = 0: nothing.
struct Tile {
    int expert, start, n, block;
};

LSMX_DEV int lane_of(int v, int l) { return __builtin_amdgcn_readlane(v, l); }

// Every expert's pairs in tiles of `height`, then those of the pairs of no
// expert, each tile `blocks` times; an expert's tiles of one block are
// neighbours, so that they share its weights, and an eighth of all of them goes
// to each XCD (workgroup b runs on XCD b % 8) so that they share its L2.  Every
// wave computes it; experts <= 1024.
LSMX_DEV Tile find_tile(const int32_t *offsets, int experts, int pairs, int height, int blocks) {
    const int lane = threadIdx.x & 63;
    const int per = (experts + 64) / 64;   // of experts + 1 entries
    const int first = lane * per;          // a lane's: first .. first + per - 1
    auto at = [&](int e) __attribute__((always_inline)) {
        const int v = offsets[min(e, experts)];
        return e > experts ? pairs : min(max(v, 0), pairs);
    };
    const int begin = at(first);
    int mine = 0, lo = begin, n0 = 0;
    for (int i = 0; i < per; ++i) {
        const int hi = at(first + i + 1), n = first + i <= experts ? max(hi - lo, 0) : 0;
        mine += (n + height - 1) / height;
        n0 = n;
        lo = hi;
    }
    const int inc = scan64(mine), all = lane_of(inc, 63) * blocks, chunk = (all + 7) / 8;
    const int unit = (int)(blockIdx.x & 7) * chunk + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= chunk || unit >= all) return Tile{0, 0, 0, 0};
    const int owner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(inc * blocks > unit));
    int left = unit - (lane_of(inc, owner) - lane_of(mine, owner)) * blocks;
    int e = owner * per, start = lane_of(begin, owner), n = lane_of(n0, owner);
    if (per > 1) {
        for (int i = 0; i < per; ++i, ++e) {
            start = __builtin_amdgcn_readfirstlane(at(e));
            n = max(__builtin_amdgcn_readfirstlane(at(e + 1)) - start, 0);
            const int units = (n + height - 1) / height * blocks;
            if (left < units) break;
            left -= units;
        }
        if (e >= owner * per + per) return Tile{0, 0, 0, 0};
    }
    const int tiles = (n + height - 1) / height;
    if (tiles == 0) return Tile{0, 0, 0, 0};
    const int block = left / tiles, m = left - block * tiles;
    if (left < 0 || block >= blocks) return Tile{0, 0, 0, 0};   // sums that passed 31 bits: no dispatch's offsets
    return Tile{e, start + m * height, min(n - m * height, height), block};
}
// Workgroups that hold every tile, whatever the offsets.
int64_t tile_units(int64_t pairs, int64_t experts, int64_t height, int64_t blocks) {
    return ((pairs / height + (experts + 1 < pairs ? experts + 1 : pairs)) * blocks + 7) / 8 * 8;
}

// The pair of row r of a tile, -1 where there is none.
LSMX_DEV int pair_at(const ExpertArgs &a, const Tile &tile, int r) {
    const uint32_t p = (uint32_t)a.order[tile.start + min(r, tile.n - 1)];
    return r < tile.n && p < (uint32_t)a.pairs ? (int)p : -1;
}
// The row of x of a tile's row r (of its last past the end).
template <bool GATED>
LSMX_DEV int64_t x_row(const ExpertArgs &a, const Tile &tile, int r) {
    const uint32_t p = (uint32_t)a.order[tile.start + min(r, tile.n - 1)], q = p < (uint32_t)a.pairs ? p : 0u;
    return GATED ? q / (uint32_t)a.k : q;
}

// g sigmoid(g) u.  exp(-g) past the type's range gives the sigmoid's 0 or 1; the
// reciprocal is within 1 step of fp32.
LSMX_DEV float silu_times(float g, float u) { return g * __builtin_amdgcn_rcpf(1.f + __expf(-g)) * u; }

// Zeros of scale 1 in elements f0 .. f0 + nf - 1 of a tile's rows.
LSMX_DEV void zero_rows(const ExpertArgs &a, const Tile &tile, int threads, int f0, int nf) {
    const int F = a.N / 2, words = nf / 4, each = words + nf / 32;
    for (int q = threadIdx.x; q < tile.n * each; q += threads) {
        const int p = pair_at(a, tile, q / each), w = q % each;
        if (p < 0) continue;
        if (w < words)
            *(uint32_t *)(a.h + (int64_t)p * F + f0 + 4 * w) = 0;
        else
            a.hs[(int64_t)p * (F / 32) + f0 / 32 + w - words] = 127;
    }
}

// ------------------------------------------------------------ few workgroups
// 8 waves for 64 rows of W (gated: 32 of the gate, the same 32 of up) and up to
// 16 pairs of one expert: the waves split K, take the weights from memory
// straight into registers, two steps of 128 at a time, and add their sums up in
// LDS.  With so few workgroups the time is one pass over K in latency: 8 waves
// a workgroup shorten it, and a ring in LDS would only lengthen it (4 experts,
// K = 2048, F = 1024: 8.3 us).
template <bool GATED>
__global__ __launch_bounds__(512) void expert_stream_kernel(ExpertArgs a) {
    constexpr int KW = 8;
    __shared__ __attribute__((aligned(16))) float sum[KW][64][16];
    __shared__ int pair_of[16];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), i16 = lane & 15, g = lane >> 4;
    const Tile tile = find_tile(a.offsets, a.experts, a.pairs, 16, (a.N + 63) / 64);
    if (tile.n == 0) return;
    const int nb = tile.block, F = a.N / 2;
    if (tile.expert == a.experts) {   // pairs of no expert: rows of zeros
        if constexpr (GATED) zero_rows(a, tile, 512, nb * 32, 32);
        return;
    }
    const int kb = a.K / 32, steps = a.K / 128, s0 = steps * wave / KW, s1 = steps * (wave + 1) / KW;
    // four tiles of 16 rows of W
    const uint8_t *wp[4], *sp[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int n0 = GATED ? nb * 32 + (r & 1) * 16 + (r >> 1) * F : nb * 64 + r * 16;
        const int64_t n = (int64_t)tile.expert * a.N + min(n0 + i16, a.N - 1);
        wp[r] = a.w + n * (a.K / 2) + 16 * g;
        sp[r] = a.ws + n * kb + g;
    }
    const int64_t row = x_row<GATED>(a, tile, i16);
    const uint8_t *xp = a.x + row * a.K + 16 * g, *xsp = a.xs + row * kb + g;
    if (t < 16) pair_of[t] = pair_at(a, tile, t);
    v4f acc[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int s = s0; s < s1; s += 2) {
        v4i w[2][4];
        v8i x[2];
        int ws[2][4], xs[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t q = min(s + u, s1 - 1);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                w[u][r] = *(const v4i *)(wp[r] + q * 64);
                ws[u][r] = sp[r][q * 4];
            }
            const v4i lo = *(const v4i *)(xp + q * 128), hi = *(const v4i *)(xp + q * 128 + 64);
            x[u] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            xs[u] = xsp[q * 4];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (s + u >= s1) continue;
            const v8i big = large_codes(x[u]), small = x[u] ^ big;
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = mfma_f4f8(w[u][r], big, acc[r], 4, 0, 0, ws[u][r], 0, xs[u]);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = mfma_f4f8(w[u][r], small, acc[r], 4, 0, 0, ws[u][r], 0, xs[u]);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[wave][r * 16 + 4 * g + q][i16] = acc[r][q];
    __syncthreads();
    auto total = [&](int r, int c) __attribute__((always_inline)) {
        float v = sum[0][r][c];
#pragma unroll
        for (int w = 1; w < KW; ++w) v += sum[w][r][c];
        return v;
    };
    if constexpr (GATED) {
        // 32 threads a pair, one element each
        const int c = t / 32, f = t % 32, p = pair_of[c];
        const float v = silu_times(total(f, c), total(32 + f, c));
        uint32_t am = f2u(v) & 0x7FFFFFFFu;
#pragma unroll
        for (int m = 1; m < 32; m *= 2) am = max(am, (uint32_t)__shfl_xor((int)am, m, 64));
        const uint32_t byte = mx8_byte(am);
        if (p >= 0) {
            a.h[(int64_t)p * F + nb * 32 + f] = (uint8_t)e4m3_x4(v * mx8_inverse(byte), 0.f, 0.f, 0.f);
            if (f == 0) a.hs[(int64_t)p * (F / 32) + nb] = (uint8_t)byte;
        }
    } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int c = t / 64 + 8 * q, n = nb * 64 + t % 64, p = pair_of[c];
            if (p >= 0 && n < a.N) a.z[(int64_t)p * a.ldz + n] = total(t % 64, c);
        }
    }
}

// ------------------------------------------------------------- LDS tiles
// A workgroup of WM * WT waves, WM along W and WT along the pairs: 256 rows of W
// (gated: of 128 elements the gate's and up's, 128 / WM of each in a wave) for
// up to BT pairs of one expert.  Stages of 128 K go straight from memory into a
// ring of three LDS slots, two stages ahead of their use: pairs' rows by the
// addresses of each lane's own row, so that nothing is gathered first.  Scales
// come four stages at a time: a load of 4 bytes a row would read as many cache
// lines each stage as the codes do.  One barrier a stage.
//
// Tiles of up to 48 pairs have four waves and half of the LDS, two workgroups a
// CU: one's loads stand under the other's products.  128 and 256 pairs, where
// an expert has them, read W less often.
template <int BT, int NW>
struct TileShape {
    static constexpr int WM = NW == 4 || BT < 256 ? 4 : 2, WT = NW / WM, NT = 64 * NW;
    static constexpr int A = 256 / WM / 16, B = BT / WT / 16;   // 16 x 16 tiles of a wave
    static constexpr int XB = BT * 128, WB = 256 * 64;          // bytes of a stage
    static constexpr int SLOT = XB + WB, ROWS = 256 + (BT < 64 ? 64 : BT);
    static constexpr int LDS = 3 * SLOT + 2 * ROWS * 16;        // and two groups of four stages' scales
    static constexpr int XL = (XB / 16 + NT - 1) / NT, WL = WB / 16 / NT, L = XL + WL;   // 16-byte loads of a thread
    static constexpr int SETS = ROWS / 64, SL = (SETS + NW - 1) / NW;   // scales
};

LSMX_DEV void dma16(const uint8_t *p, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(__builtin_amdgcn_readfirstlane(m0)) : "memory");
}

template <bool GATED, int BT, int NW>
__global__ __launch_bounds__(64 * NW, 2) void expert_tile_kernel(ExpertArgs a) {
    typedef TileShape<BT, NW> S;
    constexpr int A = S::A, B = S::B, L = S::L, G = 4;   // G: stages of a group of scales
    constexpr bool EXACT = BT == 16;   // in time that its loads leave over (at 64 pairs: 55 us, exact 83)
    __shared__ __attribute__((aligned(16))) uint8_t lds[S::LDS];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), i16 = lane & 15, g = lane >> 4;
    const int wm = wave % S::WM, wt = wave / S::WM;
    const Tile tile = find_tile(a.offsets, a.experts, a.pairs, BT, (a.N + 255) / 256);
    if (tile.n == 0) return;
    const int nb = tile.block, F = a.N / 2;
    if (tile.expert == a.experts) {
        if constexpr (GATED) zero_rows(a, tile, S::NT, nb * 128, min(128, F - nb * 128));
        return;
    }
    const int kb = a.K / 32, nk = a.K / 128;
    const int64_t first = (int64_t)tile.expert * a.N;
    // row r of the weights' tile
    auto w_row = [&](int r) __attribute__((always_inline)) {
        if constexpr (GATED) {
            constexpr int R = 128 / S::WM;   // a wave's rows of each kind
            const int f = min(nb * 128 + r / (2 * R) * R + r % R, F - 1);
            return first + f + (r / R & 1) * F;
        } else {
            return first + min(nb * 256 + r, a.N - 1);
        }
    };
    // a thread's shares of a stage.  16-byte chunk c of a pair's row lies at
    // c ^ (row & 7), of a weight's row at c ^ (row / 2 & 3): the rows that are
    // read together then cover the banks.  Where a stage's pairs are fewer than
    // the threads, several waves load the same.
    auto x_set = [&](int i) __attribute__((always_inline)) { return min(i * NW + wave, S::XB / 1024 - 1); };   // of 8 rows
    const uint8_t *xp[S::XL], *wp[S::WL], *sp[S::SL];
#pragma unroll
    for (int i = 0; i < S::XL; ++i)
        xp[i] = a.x + x_row<GATED>(a, tile, x_set(i) * 8 + lane / 8) * a.K + ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
    for (int i = 0; i < S::WL; ++i)
        wp[i] = a.w + w_row(i * 16 * NW + wave * 16 + lane / 4) * (a.K / 2) + ((lane & 3) ^ (lane >> 3 & 3)) * 16;
    // scales in sets of 64 rows: four of the weights, then the pairs'
    auto set_of = [&](int i) __attribute__((always_inline)) { return min(wave + i * NW, S::SETS - 1); };
#pragma unroll
    for (int i = 0; i < S::SL; ++i) {
        const int u = set_of(i);
        sp[i] = u < 4 ? a.ws + w_row(u * 64 + lane) * kb : a.xs + x_row<GATED>(a, tile, min((u - 4) * 64 + lane, BT - 1)) * kb;
    }
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    // load i of a stage, and the way to the next stage's: 1, or 0 past the last
    auto load = [&](int i, uint32_t slot, int step) __attribute__((always_inline)) {
        if (i < S::XL) {
            dma16(xp[i], base + slot + x_set(i) * 1024);
            xp[i] += 128 * step;
        } else {
            dma16(wp[i - S::XL], base + slot + S::XB + ((i - S::XL) * NW + wave) * 1024);
            wp[i - S::XL] += 64 * step;
        }
    };
    // the scales of the G stages from G n on, the last group's moved back to where
    // it ends with the row (nk >= 4)
    auto load_scales = [&](int n) __attribute__((always_inline)) {
        const uint32_t to = base + 3 * S::SLOT + (n & 1) * S::ROWS * 4 * G;
        const int at = min(G * n, nk - G) * 4;
#pragma unroll
        for (int i = 0; i < S::SL; ++i) dma16(sp[i] + at, to + set_of(i) * 1024);
    };
    // where stage kt's scales lie, kt = G n + i
    auto scales_of = [&](int n, int i) __attribute__((always_inline)) {
        return (uint32_t)(3 * S::SLOT + (n & 1) * S::ROWS * 4 * G + (i + max(G * n + G - nk, 0)) * 4);
    };
    int pair[B];   // of this lane's results
#pragma unroll
    for (int j = 0; j < B; ++j) pair[j] = pair_at(a, tile, (wt * B + j) * 16 + i16);
    v4f acc[A][B];
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
        for (int j = 0; j < B; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    const int x0 = (wt * B * 16 + i16) * 128 + ((g ^ (lane & 7)) << 4), w0 = S::XB + (wm * A * 16 + i16) * 64 + ((g ^ (lane >> 1 & 3)) << 4);
    const int ws0 = (wm * A * 16 + i16) * 4 * G + g, xs0 = (256 + wt * B * 16 + i16) * 4 * G + g;
    v8i x[B];
    v4i w[A];
    int xs[B], ws[A];
    auto read_x = [&](int j, uint32_t slot, uint32_t sc) __attribute__((always_inline)) {
        const uint8_t *sl = lds + slot;
        const v4i lo = *(const v4i *)(sl + x0 + j * 2048), hi = *(const v4i *)(sl + (x0 ^ 64) + j * 2048);
        x[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        xs[j] = lds[sc + xs0 + j * 64 * G];
    };
    auto read_w = [&](int i, uint32_t slot, uint32_t sc) __attribute__((always_inline)) {
        w[i] = *(const v4i *)(lds + slot + w0 + i * 1024);
        ws[i] = lds[sc + ws0 + i * 64 * G];
    };
    // products of W's tiles i0 .. i1 - 1 with pairs' tile j
    auto multiply = [&](int i0, int i1, int j) __attribute__((always_inline)) {
        const v8i big = EXACT ? large_codes(x[j]) : x[j];
#pragma unroll
        for (int i = i0; i < i1; ++i) acc[i][j] = mfma_f4f8(w[i], big, acc[i][j], 4, 0, 0, ws[i], 0, xs[j]);
        if constexpr (EXACT) {
            const v8i small = x[j] ^ big;
#pragma unroll
            for (int i = i0; i < i1; ++i) acc[i][j] = mfma_f4f8(w[i], small, acc[i][j], 4, 0, 0, ws[i], 0, xs[j]);
        }
    };
    // waits for this wave's reads and for all but its last n loads, then for the
    // other waves
    auto wait = [&](auto loads) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0x0070 | decltype(loads)::value);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    static_assert(2 * L < 16, "the count of a wait");
    load_scales(0);
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int i = 0; i < L; ++i) load(i, k * S::SLOT, k + 1 < nk);
    wait(SlotC<2 * L>{});
    if (S::WT > 1 && wt * B * 16 >= tile.n) {
        // a wave without pairs only loads: the other one of its SIMD multiplies
        uint32_t slot = 0;
        for (int kt = 0; kt < nk; ++kt) {
            wait(SlotC<L>{});
            if (kt % G == 0 && kt + G < nk) load_scales(kt / G + 1);
            const int step = kt + 4 < nk;
#pragma unroll
            for (int i = 0; i < L; ++i) load(i, slot, step);
            slot = slot == 2 * S::SLOT ? 0 : slot + S::SLOT;
        }
        wait_dma();
        return;
    }
    uint32_t sc = scales_of(0, 0);
#pragma unroll
    for (int i = 0; i < A / 2; ++i) read_w(i, 0, sc);
#pragma unroll
    for (int j = 0; j < B; ++j) read_x(j, 0, sc);
    // A stage: the pairs' rows and half of W's are in registers or on their way.
    // The other half of W is read during the first half of the products; the slot
    // is then free for the stage after the next two, whose loads go out one by
    // one between the products of the second half and of the next stage's first
    // (in one burst they keep the waves from issuing).  During the second half
    // the next stage is read, each pair's rows once their last product is issued.
    // Past the last stage the loop loads that again, and reads what it does not
    // use, without branches.
    uint32_t now = 0, before = 2 * S::SLOT;
    constexpr int L0 = L - L / 2;   // loads of the second half
    int step = 0, gn = 0, gi = 0;   // kt = G gn + gi
    for (int kt = 0; kt < nk; ++kt) {
        const uint32_t next = now == 2 * S::SLOT ? 0 : now + S::SLOT;
#pragma unroll
        for (int j = 0; j < B; ++j) {
#pragma unroll
            for (int i = A / 2 * j / B; i < A / 2 * (j + 1) / B; ++i) read_w(A / 2 + i, now, sc);
            multiply(0, A / 2, j);
            if (kt > 0)
#pragma unroll
                for (int i = L0 + L / 2 * j / B; i < L0 + L / 2 * (j + 1) / B; ++i) load(i, before, step);
            __builtin_amdgcn_sched_barrier(0);
        }
        wait(SlotC<L>{});
        step = kt + 4 < nk;
        if (gi == 0 && G * (gn + 1) < nk) load_scales(gn + 1);
        if (++gi == G) gi = 0, ++gn;
        sc = kt + 1 < nk ? scales_of(gn, gi) : sc;
#pragma unroll
        for (int i = 0; i < A / 2; ++i) read_w(i, next, sc);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < B; ++j) {
            multiply(A / 2, A, j);
            __builtin_amdgcn_sched_barrier(0);
            read_x(j, next, sc);
#pragma unroll
            for (int i = L0 * j / B; i < L0 * (j + 1) / B; ++i) load(i, now, step);
        }
        before = now;
        now = next;
    }
    wait_dma();   // nothing may land in LDS after the workgroup
#pragma unroll
    for (int j = 0; j < B; ++j) {
        const int p = pair[j];
        if constexpr (GATED) {
            // a block of 32 elements of a pair: two tiles in four lanes
#pragma unroll
            for (int b = 0; b < A / 4; ++b) {
                float v[8];
                uint32_t am = 0;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    v[q] = silu_times(acc[2 * b + q / 4][j][q % 4], acc[A / 2 + 2 * b + q / 4][j][q % 4]);
                    am = max(am, f2u(v[q]) & 0x7FFFFFFFu);
                }
                const uint32_t byte = mx8_byte(max4(am));
                const float m = mx8_inverse(byte);
                const int f = nb * 128 + wm * (A * 8) + b * 32;
                uint32_t c0 = e4m3_x4(v[0] * m, v[1] * m, v[2] * m, v[3] * m), c1 = e4m3_x4(v[4] * m, v[5] * m, v[6] * m, v[7] * m);
                neighbours(c0, c1);
                if (p >= 0 && f < F) {
                    *(uint64_t *)(a.h + (int64_t)p * F + f + 8 * g) = (uint64_t)c1 << 32 | c0;
                    if (g == 0) a.hs[(int64_t)p * (F / 32) + f / 32] = (uint8_t)byte;
                }
            }
        } else if (a.zs) {
            // rows of z in 16 bits: fp16 with a power of two for 64 elements that
            // puts the largest at 2^14 to 2^15; within 2^-11 of each down to 2^-28
            // of the largest, an eighth of bf16's own rounding
#pragma unroll
            for (int b = 0; b < A / 4; ++b) {
                uint32_t am = 0;
#pragma unroll
                for (int i = 4 * b; i < 4 * b + 4; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const uint32_t u = f2u(acc[i][j][q]) & 0x7FFFFFFFu;
                        am = max(am, u < 0x7F800000u ? u : 0u);   // infinities and NaN stay what they are
                    }
                const uint32_t e = max(max4(am) >> 23, 16u) - 14u;   // the largest below 2^15
                const float m = u2f((254u - e) << 23);
                const int n = nb * 256 + (wm * A + 4 * b) * 16;
                uint32_t o[4][2];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        typedef _Float16 v2h __attribute__((ext_vector_type(2)));
                        const v4f &v = acc[4 * b + i][j];
                        o[i][q] = __builtin_bit_cast(uint32_t, v2h{(_Float16)(v[2 * q] * m), (_Float16)(v[2 * q + 1] * m)});
                    }
#pragma unroll
                for (int i = 0; i < 4; i += 2) neighbours(o[i][0], o[i + 1][0]), neighbours(o[i][1], o[i + 1][1]);
                if (p >= 0 && n < a.N) {
                    _Float16 *z = (_Float16 *)a.z + (int64_t)p * a.ldz + n + 8 * g;   // ldz: whole eights
#pragma unroll
                    for (int i = 0; i < 4; i += 2)
                        if (n + 16 * i + 8 * g < a.N) *(v4i *)(z + 16 * i) = v4i{(int)o[i][0], (int)o[i][1], (int)o[i + 1][0], (int)o[i + 1][1]};
                    if (g == 0) a.zs[(int64_t)p * ((a.N + 63) / 64) + n / 64] = u2f(e << 23);
                }
            }
        } else if (p >= 0) {
#pragma unroll
            for (int i = 0; i < A; ++i) {
                const int n = nb * 256 + (wm * A + i) * 16 + 4 * g;
                if (n < a.N) *(v4f *)(a.z + (int64_t)p * a.ldz + n) = acc[i][j];
            }
        }
    }
}

// y_t = sum_j weight_tj z_tj over the pairs that have an expert, in the order of
// their slots, in fp32; 8 elements a thread.  Sums by atomics in the products'
// epilogue would need no z, but their order, and the result, would change.  z is
// read once, past the caches (combine of 8192 tokens of 128 experts 160 -> 156 us;
// stores past them too were slower, 167).
template <int DT, bool HALF>
__global__ __launch_bounds__(256) void expert_join_kernel(ExpertArgs a) {
    typedef typename Elem<DT>::S S;
    const int chunks = (a.N + 7) / 8, blocks = (chunks + 255) / 256;
    const int64_t token = blockIdx.x / blocks;
    const int n = ((blockIdx.x % blocks) * 256 + threadIdx.x) * 8;
    if (n >= a.N) return;
    float v[8] = {};
#pragma unroll 4
    for (int j = 0; j < a.k; ++j) {
        const int64_t p = token * a.k + j;
        if ((uint32_t)a.ids[p] >= (uint32_t)a.experts) continue;
        if constexpr (HALF) {
            const float w = a.weights[p], scale = a.zs[p * ((a.N + 63) / 64) + n / 64];
            typedef _Float16 v8h __attribute__((ext_vector_type(8)));
            const v8h z = __builtin_nontemporal_load((const v8h *)((const _Float16 *)a.z + p * a.ldz + n));
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += w * ((float)z[i] * scale);
        } else {
            const float w = a.weights[p];
            const v4f *q = (const v4f *)(a.z + p * a.ldz + n);
            const v4f z0 = __builtin_nontemporal_load(q), z1 = __builtin_nontemporal_load(q + 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += w * z0[i], v[4 + i] += w * z1[i];
        }
    }
    S *y = (S *)a.y + token * a.N + n;
    typedef S V __attribute__((ext_vector_type(8), aligned(16)));
    if (a.N % 8 == 0 && (uintptr_t)a.y % 16 == 0) {
        V o;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = Elem<DT>::store(v[i]);
        *(V *)y = o;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (n + i < a.N) y[i] = Elem<DT>::store(v[i]);
    }
}

template <bool GATED>
hipError_t stream(const ExpertArgs &a, hipStream_t s) {
    expert_stream_kernel<GATED><<<(unsigned)tile_units(a.pairs, a.experts, 16, (a.N + 63) / 64), 512, 0, s>>>(a);
    return hipGetLastError();
}
template <bool GATED, int BT, int NW>
hipError_t tiles(const ExpertArgs &a, hipStream_t s) {
    expert_tile_kernel<GATED, BT, NW><<<(unsigned)tile_units(a.pairs, a.experts, BT, (a.N + 255) / 256), 64 * NW, 0, s>>>(a);
    return hipGetLastError();
}
// Pairs of a tile, or 0 for the stream kernel.  us at 32 experts, K = 2048,
// F = 1024, by pairs an expert (gated; combine, its K = 1024, alike):
//            1     4     8    24    48    96   128   256   512  1024
//   stream  14.3  26.3  31.7
//     16    12.7  15.3  20.0  29.6  33.1  53.3
//     32    11.9  14.5  14.9  19.4  28.4  32.6  40.2
//     48    12.9  15.2  15.5  21.5  21.9  30.0  39.1  55.1  107   226
//    128    13.4  15.3  15.7  20.2  30.3  35.0  35.1  55.1   90.7 191
//    256    18.3  19.8  19.9  21.7  28.8  46.5  45.4  58.0   88.2 153
// and with 128 experts, where the weights do not stay in the caches:
//     16    26.7  45.1  53.9  81.5 128
//     32    26.4  44.9  47.2  61.5  85.3
//     48    27.1  45.9  47.6  58.2  77.6 113.5 136   258   446   814
//    128    31.9  54.6  56.8  64.3  82.1 110.1 132   206   362   671
//    256    39.1  71.4  72.0  75.1  88.5 116.4 131   188   322   575
// Pairs are not spread evenly; 16 where it costs little, for its exact products.
int height_of(const ExpertArgs &a) {
    // a tile needs two groups' worth of stages; up to 384 workgroups, more waves
    // for each (4 pairs, K = 2048, F = 1024: 8.3 against 10.0 us)
    if (a.K < 512 || (int64_t)a.pairs * ((a.N + 63) / 64) <= 384) return 0;
    const int64_t per = a.pairs / a.experts;
    if (per <= 96) return per <= 4 ? 16 : per <= 24 ? 32 : 48;
    // full tiles, or as many as fill the 256 CUs three times
    const int64_t units = (a.pairs / 256 + a.experts / 2) * ((a.N + 255) / 256);
    return per > 400 || units >= 768 ? 256 : 128;
}
template <bool GATED>
hipError_t products(const ExpertArgs &a, int height, hipStream_t s) {
    switch (height) {
        case 16: return tiles<GATED, 16, 4>(a, s);
        case 32: return tiles<GATED, 32, 4>(a, s);
        case 48: return tiles<GATED, 48, 4>(a, s);
        case 128: return tiles<GATED, 128, 8>(a, s);
        case 256: return tiles<GATED, 256, 8>(a, s);
        default: return stream<GATED>(a, s);
    }
}

template <int DT>
hipError_t join(const ExpertArgs &a, hipStream_t s) {
    const int64_t chunks = (a.N + 7) / 8, grid = (chunks + 255) / 256 * a.tokens;
    if (a.zs)
        expert_join_kernel<DT, true><<<(unsigned)grid, 256, 0, s>>>(a);
    else
        expert_join_kernel<DT, false><<<(unsigned)grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_expert_gated(const ExpertArgs &a, hipStream_t s) { return products<true>(a, height_of(a), s); }

hipError_t launch_expert_combine(const ExpertArgs &a0, hipStream_t s) {
    ExpertArgs a = a0;
    const int height = height_of(a);
    // bf16 sums of many rows take the pairs' rows in 16 bits.  us with them in 32
    // and in 16, 128 experts, K = 1024, N = 2048, by pairs an expert:
    //   32 45.7 43.9   48 53.7 51.8   96 97.3 76.8   192 164 145   512 409 318
    if (a.y_dtype == LSMX_BF16 && height >= 48) a.zs = (float *)((uint8_t *)a.z + (int64_t)a.pairs * a.ldz * 2);
    const hipError_t e = products<false>(a, height, s);
    if (e != hipSuccess) return e;
    return a.y_dtype == LSMX_F32 ? join<LSMX_F32>(a, s) : a.y_dtype == LSMX_BF16 ? join<LSMX_BF16>(a, s) : join<LSMX_F16>(a, s);
}

}  // namespace lsmx
