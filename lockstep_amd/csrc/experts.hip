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
#include "lsmx_dma.h"
#include "lsmx_internal.h"

namespace lsmx {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

__device__ v4f mfma_f4f8(v4i a, v8i b, v4f c, int cbsz, int blgp, int opsel_a, int scale_a, int opsel_b, int scale_b)
    __asm("llvm.amdgcn.mfma.scale.f32.16x16x128.f8f6f4.v4i32.v8i32");

namespace {

// What a workgroup does: block `block` of W's rows for the pairs
// order[start .. start + n), all of expert `expert`, or of no expert where that
// is `experts`.  n = 0: nothing.
struct Tile {
    int expert, start, n, block;
};

// Every expert's pairs in tiles of `height`, then those of the pairs of no
// expert, each tile `blocks` times; an expert's tiles of one block are
// neighbours, so that they share its weights, and an eighth of all of them goes
// to each XCD (workgroup b runs on XCD b % 8) so that they share its L2.  Every
// wave computes it; experts <= 1024.
LSMX_DEV Tile find_tile(const int32_t *offsets, int experts, int pairs, int height, int blocks) {
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
    const int all = __builtin_amdgcn_readlane(inc, 63) * blocks, chunk = (all + 7) / 8;
    const int unit = (int)(blockIdx.x & 7) * chunk + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= chunk || unit >= all) return Tile{0, 0, 0, 0};
    const int owner = __builtin_ctzll(__builtin_amdgcn_ballot_w64(inc * blocks > unit));
    int left = unit - (__builtin_amdgcn_readlane(inc, owner) - __builtin_amdgcn_readlane(mine, owner)) * blocks;
    int e = owner * per;
    for (int i = 0; i < per; ++i, ++e) {
        const int lo2 = at(e), n = max(at(e + 1) - lo2, 0), tiles = (n + height - 1) / height;
        if (left < tiles * blocks) {
            const int m = left % tiles;
            return Tile{e, lo2 + m * height, min(n - m * height, height), left / tiles};
        }
        left -= tiles * blocks;
    }
    return Tile{0, 0, 0, 0};
}
// Workgroups that hold every tile, whatever the offsets.
int64_t tile_units(int64_t pairs, int64_t experts, int64_t height, int64_t blocks) {
    return ((pairs / height + (experts + 1 < pairs ? experts + 1 : pairs)) * blocks + 7) / 8 * 8;
}

// g sigmoid(g) u.  exp(-g) past the type's range gives the sigmoid's 0 or 1; the
// reciprocal is within 1 step of fp32.
LSMX_DEV float silu_times(float g, float u) { return g * __builtin_amdgcn_rcpf(1.f + __expf(-g)) * u; }

// Zeros of scale 1 in elements f0 .. f0 + nf - 1 of the rows of n pairs.
template <int NT, typename P>
LSMX_DEV void zero_rows(const ExpertArgs &a, const P &pair_of, int n, int f0, int nf) {
    const int F = a.N / 2, words = nf / 4, each = words + nf / 32;
    for (int q = threadIdx.x; q < n * each; q += NT) {
        const int p = pair_of(q / each), w = q % each;
        if (p < 0) continue;
        if (w < words)
            *(uint32_t *)(a.h + (int64_t)p * F + f0 + 4 * w) = 0;
        else
            a.hs[(int64_t)p * (F / 32) + f0 / 32 + w - words] = 127;
    }
}

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
    const Tile tile = find_tile(a.offsets, a.experts, a.pairs, C, (a.N + 63) / 64);
    const int nb = tile.block;
    if (tile.n == 0) return;
    if (t < C) {
        const uint32_t p = t < tile.n ? (uint32_t)a.order[tile.start + t] : 0xFFFFFFFFu;
        pair_of[t] = p < (uint32_t)a.pairs ? (int)p : -1;
    }
    __syncthreads();
    const int F = a.N / 2;
    if (tile.expert == a.experts) {   // pairs of no expert: rows of zeros
        if constexpr (GATED) zero_rows<64 * KW>(a, [&](int r) { return pair_of[r]; }, tile.n, nb * 32, 32);
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

// ------------------------------------------------------------ many rows
// A workgroup of 8 waves, WM along W and 8 / WM along the pairs: 256 rows of W
// (gated: of 128 elements the gate's and up's, 256 / WM / 2 of each in a wave)
// for up to BT pairs of one expert.  Stages of 128 K go straight from memory
// into a ring of three LDS slots, two stages ahead of their use: pairs' rows
// by the addresses of each lane's own row, so that nothing is gathered first.
// One barrier a stage: after it the stage is there for every wave, and the slot
// of the stage before is free.
template <int BT>
struct TileShape {
    static constexpr int WM = BT == 256 ? 2 : 4, WT = 8 / WM;
    static constexpr int A = 256 / WM / 16, B = BT / WT / 16;   // 16 x 16 tiles of a wave
    static constexpr int XB = BT * 128, WB = 256 * 64;          // bytes of a stage
    static constexpr int SLOT = XB + WB, ROWS = BT + 256;
    static constexpr int LDS = 3 * SLOT + 2 * ROWS * 16;        // and two groups of 4 stages' scales
    static constexpr int XL = XB / 16 / 512;                    // 16-byte loads of a thread
};

LSMX_DEV void dma16(const uint8_t *p, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(__builtin_amdgcn_readfirstlane(m0)) : "memory");
}
LSMX_DEV void dma4(const uint8_t *p, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(__builtin_amdgcn_readfirstlane(m0)) : "memory");
}

template <bool GATED, int BT>
__global__ __launch_bounds__(512, 2) void expert_tile_kernel(ExpertArgs a) {
    typedef TileShape<BT> S;
    constexpr int A = S::A, B = S::B;
    __shared__ __attribute__((aligned(16))) uint8_t lds[S::LDS];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), i16 = lane & 15, g = lane >> 4;
    const int wm = wave % S::WM, wt = wave / S::WM;
    const int F = a.N / 2;
    const Tile tile = find_tile(a.offsets, a.experts, a.pairs, BT, (a.N + 255) / 256);
    const int nb = tile.block;
    if (tile.n == 0) return;
    // the pair of row r of the tile, -1 past the last
    auto pair_of = [&](int r) __attribute__((always_inline)) {
        const uint32_t p = r < tile.n ? (uint32_t)a.order[tile.start + r] : 0xFFFFFFFFu;
        return p < (uint32_t)a.pairs ? (int)p : -1;
    };
    if (tile.expert == a.experts) {
        if constexpr (GATED) zero_rows<512>(a, pair_of, tile.n, nb * 128, min(128, F - nb * 128));
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
    auto x_row = [&](int r) __attribute__((always_inline)) {
        const int p = max(pair_of(min(r, tile.n - 1)), 0);
        return (int64_t)(GATED ? p / a.k : p);
    };
    // a thread's shares of a stage.  16-byte chunk c of a pair's row lies at
    // c ^ (row & 7), of a weight's row at c ^ (row / 2 & 3): the rows that are
    // read together then cover the banks.
    const uint8_t *xp[S::XL], *wp[2], *sp;
#pragma unroll
    for (int i = 0; i < S::XL; ++i) xp[i] = a.x + x_row(i * 64 + wave * 8 + lane / 8) * a.K + ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        wp[i] = a.w + w_row(i * 128 + wave * 16 + lane / 4) * (a.K / 2) + ((lane & 3) ^ (lane >> 3 & 3)) * 16;
    // scales, 16 bytes a row for four stages: waves 0 .. 3 the weights', the
    // others the pairs'
    if (wave < 4)
        sp = a.ws + w_row(wave * 64 + lane) * kb;
    else
        sp = a.xs + x_row(min((wave - 4) * 64 + lane, BT - 1)) * kb;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    constexpr int L = S::XL + 2;   // loads of a stage
    // load i of a stage, and the way to the next stage's: 1, or 0 past the last
    auto load = [&](int i, uint32_t slot, int step) __attribute__((always_inline)) {
        if (i < S::XL) {
            dma16(xp[i], base + slot + (i * 8 + wave) * 1024);
            xp[i] += 128 * step;
        } else {
            dma16(wp[i - S::XL], base + slot + S::XB + ((i - S::XL) * 8 + wave) * 1024);
            wp[i - S::XL] += 64 * step;
        }
    };
    // the scales of stages 4 n .. 4 n + 3, the last group's moved back to where
    // it ends with the row (nk >= 4)
    auto group = [&](int n) __attribute__((always_inline)) { return min(4 * n, nk - 4); };
    auto load_scales = [&](int n) __attribute__((always_inline)) {
        if (wave < 4 + BT / 64) dma16(sp + group(n) * 4, base + 3 * S::SLOT + (n & 1) * S::ROWS * 16 + wave * 1024);
    };
    auto scales_of = [&](int kt) __attribute__((always_inline)) {
        return (uint32_t)(3 * S::SLOT + (kt >> 2 & 1) * S::ROWS * 16 + (kt - group(kt >> 2)) * 4);
    };
    v4f acc[A][B];
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
        for (int j = 0; j < B; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    const int x0 = (wt * B * 16 + i16) * 128 + ((g ^ (lane & 7)) << 4), w0 = S::XB + (wm * A * 16 + i16) * 64 + ((g ^ (lane >> 1 & 3)) << 4);
    const int ws0 = (wm * A * 16 + i16) * 16 + g, xs0 = (256 + wt * B * 16 + i16) * 16 + g;
    v8i x[B];
    v4i w[A];
    int xs[B], ws[A];
    auto read_x = [&](int j, uint32_t slot, uint32_t sc) __attribute__((always_inline)) {
        const uint8_t *sl = lds + slot;
        const v4i lo = *(const v4i *)(sl + x0 + j * 2048), hi = *(const v4i *)(sl + (x0 ^ 64) + j * 2048);
        x[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        xs[j] = lds[sc + xs0 + j * 256];
    };
    auto read_w = [&](int i, uint32_t slot, uint32_t sc) __attribute__((always_inline)) {
        w[i] = *(const v4i *)(lds + slot + w0 + i * 1024);
        ws[i] = lds[sc + ws0 + i * 256];
    };
    // waits for this wave's reads and for all but its last n loads, then for the
    // other waves
    auto wait = [&](auto loads) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0x0070 | decltype(loads)::value);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    load_scales(0);
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int i = 0; i < L; ++i) load(i, k * S::SLOT, k + 1 < nk);
    wait(SlotC<2 * L>{});
    uint32_t sc = scales_of(0);
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
    // The loop has no branches: past the last stage it loads that again, and
    // reads what it does not use.
    uint32_t now = 0, before = 2 * S::SLOT;
    constexpr int L0 = L - L / 2;   // loads of the second half
    int step = 0;
    for (int kt = 0; kt < nk; ++kt) {
        const uint32_t next = now == 2 * S::SLOT ? 0 : now + S::SLOT;
#pragma unroll
        for (int j = 0; j < B; ++j) {
#pragma unroll
            for (int i = A / 2 * j / B; i < A / 2 * (j + 1) / B; ++i) read_w(A / 2 + i, now, sc);
#pragma unroll
            for (int i = 0; i < A / 2; ++i) acc[i][j] = mfma_f4f8(w[i], x[j], acc[i][j], 4, 0, 0, ws[i], 0, xs[j]);
            if (kt > 0)
#pragma unroll
                for (int i = L0 + L / 2 * j / B; i < L0 + L / 2 * (j + 1) / B; ++i) load(i, before, step);
            __builtin_amdgcn_sched_barrier(0);
        }
        wait(SlotC<L>{});
        step = kt + 4 < nk;
        sc = scales_of(min(kt + 1, nk - 1));
        if ((kt & 3) == 0 && kt + 4 < nk) load_scales(kt / 4 + 1);
#pragma unroll
        for (int i = 0; i < A / 2; ++i) read_w(i, next, sc);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < B; ++j) {
#pragma unroll
            for (int i = A / 2; i < A; ++i) acc[i][j] = mfma_f4f8(w[i], x[j], acc[i][j], 4, 0, 0, ws[i], 0, xs[j]);
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
        const int p = pair_of((wt * B + j) * 16 + i16);
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
                am = max(am, (uint32_t)__shfl_xor((int)am, 16, 64));
                am = max(am, (uint32_t)__shfl_xor((int)am, 32, 64));
                const uint32_t byte = mx8_byte(am);
                const float m = mx8_inverse(byte);
                const int f = nb * 128 + wm * (A * 8) + b * 32;
                if (p >= 0 && f < F) {
                    uint8_t *h = a.h + (int64_t)p * F + f + 4 * g;
                    *(uint32_t *)h = e4m3_x4(v[0] * m, v[1] * m, v[2] * m, v[3] * m);
                    *(uint32_t *)(h + 16) = e4m3_x4(v[4] * m, v[5] * m, v[6] * m, v[7] * m);
                    if (g == 0) a.hs[(int64_t)p * (F / 32) + f / 32] = (uint8_t)byte;
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
    const int64_t units = tile_units(a.pairs, a.experts, 16 * NT, (a.N + 63) / 64);
    expert_stream_kernel<GATED, NT, KW><<<(unsigned)units, 64 * KW, 0, s>>>(a);
    return hipGetLastError();
}
template <bool GATED, int BT>
hipError_t tiles(const ExpertArgs &a, hipStream_t s) {
    const int64_t units = tile_units(a.pairs, a.experts, BT, (a.N + 255) / 256);
    expert_tile_kernel<GATED, BT><<<(unsigned)units, 512, 0, s>>>(a);
    return hipGetLastError();
}
template <bool GATED>
hipError_t products(const ExpertArgs &a, hipStream_t s) {
    if (a.K < 512) return stream<GATED, 1, 8>(a, s);
    const int64_t per = a.pairs / a.experts;
    return per <= 8 ? stream<GATED, 1, 8>(a, s) : per <= 32 ? stream<GATED, 4, 4>(a, s) : per <= 256 ? tiles<GATED, 128>(a, s) : tiles<GATED, 256>(a, s);
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
