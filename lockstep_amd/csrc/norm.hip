// Root-mean-square norm with the residual's addition, forward and backward.
//
//   h = round(x + r),  inv = (mean(h^2) + eps)^-1/2,  y = h inv w
//   dx = dr = inv (g - h inv^2 mean(g h)) + dh  with g = dy w;  dw = sum over rows of dy h inv
//
// Forward and backward read each operand once: a row stays in the registers
// of the threads that hold it (fp32) between the sum of squares and the
// output.  Sums are fp32; they have one order, so results do not depend on
// the run.  Memory bound: 8192 rows of 8192 in bf16 with a residual and MXFP8
// in 107 us (5.7 TB/s; a large copy makes 4.9), backward with dw of 8190 rows of
// 4096 in fp16 42 us.
#include "lsmx_block.h"

namespace lsmx {

namespace {

// Vectors of VEC elements: 16-byte loads of 8 16-bit elements (two of 4 fp32
// ones), or single elements where rows are not aligned.
template <int DT, int VEC>
struct Vec {
    typedef typename Elem<DT>::S S;
    typedef S V __attribute__((ext_vector_type(VEC), aligned(VEC * sizeof(S) < 16 ? VEC * sizeof(S) : 16)));
    static LSMX_DEV void load(const S *p, float (&f)[VEC]) {
        if constexpr (VEC == 1) {
            f[0] = Elem<DT>::load(*p);
        } else {
            const V v = *(const V *)p;
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = Elem<DT>::load(v[i]);
        }
    }
    static LSMX_DEV void store(S *p, const float (&f)[VEC]) {
        if constexpr (VEC == 1) {
            *p = Elem<DT>::store(f[0]);
        } else {
            V v;
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = Elem<DT>::store(f[i]);
            *(V *)p = v;
        }
    }
};

template <int DT, int VEC>
LSMX_DEV void load_w(const void *w, int w_dtype, int64_t at, float (&f)[VEC]) {
    if (w_dtype == LSMX_F32)
        Vec<LSMX_F32, VEC>::load((const float *)w + at, f);
    else
        Vec<DT, VEC>::load((const typename Elem<DT>::S *)w + at, f);
}

// Sum over the TPR threads of a row; in every thread of the row.  `red` holds
// one float per wave; `slot` alternates so that one barrier a sum is enough.
LSMX_DEV float wave_sum(float v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m, 64);
    return v;
}
template <int TPR>
LSMX_DEV float row_sum(float v, float *red) {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v += red[i];
    }
    return v;
}

// The MXFP8 codes and scale of 8 elements a thread, a block of 32 in 4 threads.
LSMX_DEV void store_mx8(const float (&y)[8], uint8_t *codes, uint8_t *scale, int64_t at) {
    uint32_t am = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) am = max(am, f2u(y[i]) & 0x7FFFFFFFu);
    am = max(am, (uint32_t)__shfl_xor((int)am, 1, 64));
    am = max(am, (uint32_t)__shfl_xor((int)am, 2, 64));
    const uint32_t byte = mx8_byte(am);
    const float m = mx8_inverse(byte);
    uint2 c;
    c.x = e4m3_x4(y[0] * m, y[1] * m, y[2] * m, y[3] * m);
    c.y = e4m3_x4(y[4] * m, y[5] * m, y[6] * m, y[7] * m);
    *(uint2 *)(codes + at) = c;
    if ((threadIdx.x & 3) == 0) scale[at / 32] = (uint8_t)byte;
}

// A row in TPR threads of NV vectors each.  NV = 0: rows of any length, the
// sum of squares from a first pass and the output from a second one over what
// it wrote (or over x where there is no residual).
template <int DT, int VEC, int NV, int TPR>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_fwd_kernel(NormArgs a) {
    typedef typename Elem<DT>::S S;
    constexpr int NT = TPR < 256 ? 256 : TPR;
    __shared__ float red[NT / 64];
    const int tid = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
    if (row >= a.rows) return;  // TPR < 256 only: no barrier follows there
    const S *x = (const S *)a.x + row * a.ldx, *r = (const S *)a.r + row * a.ldr;
    S *h = (S *)a.h + row * a.dim, *y = (S *)a.y + row * a.dim;
    const float inv_dim = 1.f / (float)a.dim;
    auto sum_of = [&](int64_t at, float (&f)[VEC]) __attribute__((always_inline)) {
        Vec<DT, VEC>::load(x + at, f);
        if (a.r) {
            float g[VEC];
            Vec<DT, VEC>::load(r + at, g);
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = Elem<DT>::load(Elem<DT>::store(f[i] + g[i]));
            Vec<DT, VEC>::store(h + at, f);
        }
    };
    auto finish = [&](int64_t at, float inv, const float (&f)[VEC]) __attribute__((always_inline)) {
        float w[VEC], o[VEC];
        load_w<DT, VEC>(a.w, a.w_dtype, at, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = f[i] * inv * w[i];
        Vec<DT, VEC>::store(y + at, o);
        if constexpr (VEC == 8)
            if (a.codes) store_mx8(o, a.codes, a.scale, row * a.dim + at);
    };
    float ss = 0.f;
    if constexpr (NV > 0) {
        float f[NV][VEC];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t at = (int64_t)(tid + TPR * j) * VEC;
            if (at < a.dim) {
                sum_of(at, f[j]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) ss += f[j][i] * f[j][i];
            }
        }
        const float inv = rsqrtf(row_sum<TPR>(ss, red) * inv_dim + a.eps);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t at = (int64_t)(tid + TPR * j) * VEC;
            if (at < a.dim) finish(at, inv, f[j]);
        }
    } else {
        for (int64_t at = (int64_t)tid * VEC; at < a.dim; at += (int64_t)TPR * VEC) {
            float f[VEC];
            sum_of(at, f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) ss += f[i] * f[i];
        }
        const float inv = rsqrtf(row_sum<TPR>(ss, red) * inv_dim + a.eps);
        const S *from = a.r ? h : x;  // a thread reads back what it wrote itself
        for (int64_t at = (int64_t)tid * VEC; at < a.dim; at += (int64_t)TPR * VEC) {
            float f[VEC];
            Vec<DT, VEC>::load(from + at, f);
            finish(at, inv, f);
        }
    }
}

// Two sums over a row at once.
template <int TPR>
LSMX_DEV void row_sum2(float &u, float &v, float (*red)[TPR / 64 > 0 ? TPR / 64 : 1]) {
    u = wave_sum(u), v = wave_sum(v);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = u, red[1][threadIdx.x >> 6] = v;
        __syncthreads();
        u = v = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) u += red[0][i], v += red[1][i];
        __syncthreads();
    }
}

// Backward: a workgroup of TPR threads takes the rows blockIdx.x, + gridDim.x,
// ..; its share of dw stays in the registers until the end, so that the shares
// cost gridDim.x rows of fp32 in all.  NV = 0: rows of any length, two passes
// over h and dy, dw's shares added up in memory (a thread's own elements).
template <int DT, int VEC, int NV, int TPR>
__global__ __launch_bounds__(TPR) void norm_bwd_kernel(NormBwdArgs a) {
    typedef typename Elem<DT>::S S;
    __shared__ float red[2][TPR / 64];
    constexpr int N = NV > 0 ? NV : 1;
    const int tid = threadIdx.x;
    const float inv_dim = 1.f / (float)a.dim;
    float acc[N][VEC] = {};
    float *part = a.part + (int64_t)blockIdx.x * a.dim;
    auto finish = [&](int64_t at, int64_t row, const float (&h)[VEC], const float (&d)[VEC], const float (&w)[VEC], float inv,
                      float c) __attribute__((always_inline)) {
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = inv * (d[i] * w[i] - h[i] * c);
        if (a.dh) {
            float e[VEC];
            Vec<DT, VEC>::load((const S *)a.dh + row * a.lddh + at, e);
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] += e[i];
        }
        Vec<DT, VEC>::store((S *)a.dx + row * a.dim + at, o);
    };
    if constexpr (NV == 0) {
        if (a.dw)
            for (int64_t at = (int64_t)tid * VEC; at < a.dim; at += (int64_t)TPR * VEC)
                for (int i = 0; i < VEC; ++i) part[at + i] = 0.f;
    }
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const S *hp = (const S *)a.h + row * a.ldh, *dp = (const S *)a.dy + row * a.lddy;
        float ss = 0.f, gh = 0.f;
        if constexpr (NV > 0) {
            float h[N][VEC], d[N][VEC], w[N][VEC];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t at = (int64_t)(tid + TPR * j) * VEC;
                if (at < a.dim) {
                    Vec<DT, VEC>::load(hp + at, h[j]);
                    Vec<DT, VEC>::load(dp + at, d[j]);
                    load_w<DT, VEC>(a.w, a.w_dtype, at, w[j]);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) ss += h[j][i] * h[j][i], gh += d[j][i] * w[j][i] * h[j][i];
                }
            }
            row_sum2<TPR>(ss, gh, red);
            const float inv = rsqrtf(ss * inv_dim + a.eps), c = gh * inv_dim * inv * inv;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t at = (int64_t)(tid + TPR * j) * VEC;
                if (at < a.dim) {
                    finish(at, row, h[j], d[j], w[j], inv, c);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[j][i] += d[j][i] * h[j][i] * inv;
                }
            }
        } else {
            for (int64_t at = (int64_t)tid * VEC; at < a.dim; at += (int64_t)TPR * VEC) {
                float h[VEC], d[VEC], w[VEC];
                Vec<DT, VEC>::load(hp + at, h);
                Vec<DT, VEC>::load(dp + at, d);
                load_w<DT, VEC>(a.w, a.w_dtype, at, w);
#pragma unroll
                for (int i = 0; i < VEC; ++i) ss += h[i] * h[i], gh += d[i] * w[i] * h[i];
            }
            row_sum2<TPR>(ss, gh, red);
            const float inv = rsqrtf(ss * inv_dim + a.eps), c = gh * inv_dim * inv * inv;
            for (int64_t at = (int64_t)tid * VEC; at < a.dim; at += (int64_t)TPR * VEC) {
                float h[VEC], d[VEC], w[VEC];
                Vec<DT, VEC>::load(hp + at, h);
                Vec<DT, VEC>::load(dp + at, d);
                load_w<DT, VEC>(a.w, a.w_dtype, at, w);
                finish(at, row, h, d, w, inv, c);
                if (a.dw)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) part[at + i] += d[i] * h[i] * inv;
            }
        }
    }
    if constexpr (NV > 0) {
        if (a.dw)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t at = (int64_t)(tid + TPR * j) * VEC;
                if (at < a.dim) Vec<LSMX_F32, VEC>::store(part + at, acc[j]);
            }
    }
}

// dw: the shares of `groups` workgroups added up, 16 columns a workgroup, its 64
// sets of 16 lanes every 64th share each.
template <int DT>
__global__ __launch_bounds__(1024) void norm_dw_kernel(const float *part, int groups, int64_t dim, void *dw) {
    __shared__ float red[16][16];
    const int c = threadIdx.x & 15, set = threadIdx.x >> 4;
    const int64_t col = (int64_t)blockIdx.x * 16 + c;
    float s = 0.f;
    if (col < dim)
#pragma unroll 4
        for (int g = set; g < groups; g += 64) s += part[g * dim + col];
    s += __shfl_xor(s, 16, 64);
    s += __shfl_xor(s, 32, 64);
    if ((threadIdx.x & 63) < 16) red[threadIdx.x >> 6][c] = s;
    __syncthreads();
    if (threadIdx.x < 16 && col < dim) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += red[i][c];
        ((typename Elem<DT>::S *)dw)[col] = Elem<DT>::store(s);
    }
}

template <int DT, int VEC, int NV, int TPR>
hipError_t fwd(const NormArgs &a, hipStream_t s) {
    constexpr int NT = TPR < 256 ? 256 : TPR;
    norm_fwd_kernel<DT, VEC, NV, TPR><<<(unsigned)((a.rows + NT / TPR - 1) / (NT / TPR)), NT, 0, s>>>(a);
    return hipGetLastError();
}
template <int DT, int VEC, int NV, int TPR>
hipError_t bwd(const NormBwdArgs &a, hipStream_t s) {
    norm_bwd_kernel<DT, VEC, NV, TPR><<<(unsigned)norm_bwd_groups(a.rows), TPR, 0, s>>>(a);
    return hipGetLastError();
}

bool rows_of_vectors(const void *p, int64_t ld, int64_t dim, int dtype) {
    const int64_t b = dtype == LSMX_F32 ? 4 : 2;
    return dim % 8 == 0 && (reinterpret_cast<uintptr_t>(p) % 16) == 0 && (ld * b) % 16 == 0;
}

// Threads and vectors a row.  A row in more threads is done sooner, which counts
// for few rows; many rows hide one another's latency, and threads of several
// vectors have fewer barriers and sums.  us in bf16 with a residual and MXFP8:
//   dim   rows    1024x1  512x2  512x1  256x4  256x2  256x1  64x2
//   1024     8                                           2.5    3.3
//          512                                           2.9    3.7
//         8192                                          14.7   13.2
//   4096     8                    2.7            3.5
//          512                    4.5            5.0
//         8192                   52.5           51.0
//   8192     8       3.1    3.5           5.1
//          512       7.5    7.3           8.2
//         2048      24.8   23.8          23.0
//         8192     107    112            121
// and 16384: 1024x2 24.0 and 219 us (1024, 8192 rows), 1024x4 26.2 and 229.
template <int DT>
hipError_t fwd_of(const NormArgs &a, hipStream_t s) {
    const bool vec = rows_of_vectors(a.x, a.ldx, a.dim, DT) && (!a.r || rows_of_vectors(a.r, a.ldr, a.dim, DT)) &&
                     rows_of_vectors(a.w, 0, a.dim, a.w_dtype) && rows_of_vectors(a.y, a.dim, a.dim, DT) &&
                     rows_of_vectors(a.h, a.dim, a.dim, DT);
    if (vec) {
        if (a.dim <= 512) return fwd<DT, 8, 1, 64>(a, s);
        if (a.dim <= 1024 && a.rows >= 2048) return fwd<DT, 8, 2, 64>(a, s);
        if (a.dim <= 2048) return fwd<DT, 8, 1, 256>(a, s);
        if (a.dim <= 4096) return a.rows <= 512 ? fwd<DT, 8, 1, 512>(a, s) : fwd<DT, 8, 2, 256>(a, s);
        // few rows, or more than the caches hold
        if (a.dim <= 8192) return a.rows <= 256 || a.rows > 4096 ? fwd<DT, 8, 1, 1024>(a, s) : fwd<DT, 8, 2, 512>(a, s);
        if (a.dim <= 16384) return fwd<DT, 8, 2, 1024>(a, s);
        if (a.dim <= 32768) return fwd<DT, 8, 4, 1024>(a, s);
        return fwd<DT, 8, 0, 1024>(a, s);
    }
    if (a.dim <= 512) return fwd<DT, 1, 8, 64>(a, s);
    if (a.dim <= 2048) return fwd<DT, 1, 8, 256>(a, s);
    if (a.dim <= 8192) return fwd<DT, 1, 32, 256>(a, s);
    return fwd<DT, 1, 0, 1024>(a, s);
}

// The same for the backward pass, whose workgroups keep dw's share besides.  us
// of 8192 rows with dh and dw in bf16: 4096 256x2 42.0, 512x1 43.2; 8192 512x2
// 94.5, 1024x1 117, 256x4 124; 16384 1024x2 202, two passes 376; of 512 rows of
// 32768 two passes 72, 1024x4 88.
template <int DT>
hipError_t bwd_of(const NormBwdArgs &a, hipStream_t s) {
    const bool vec = rows_of_vectors(a.h, a.ldh, a.dim, DT) && rows_of_vectors(a.dy, a.lddy, a.dim, DT) &&
                     (!a.dh || rows_of_vectors(a.dh, a.lddh, a.dim, DT)) && rows_of_vectors(a.w, 0, a.dim, a.w_dtype) &&
                     rows_of_vectors(a.dx, a.dim, a.dim, DT) && rows_of_vectors(a.part, 0, a.dim, LSMX_F32);
    if (vec) {
        if (a.dim <= 2048) return bwd<DT, 8, 1, 256>(a, s);
        if (a.dim <= 4096) return bwd<DT, 8, 2, 256>(a, s);
        if (a.dim <= 8192) return bwd<DT, 8, 2, 512>(a, s);
        if (a.dim <= 16384) return bwd<DT, 8, 2, 1024>(a, s);
        return bwd<DT, 8, 0, 1024>(a, s);
    }
    if (a.dim <= 2048) return bwd<DT, 1, 8, 256>(a, s);
    if (a.dim <= 8192) return bwd<DT, 1, 32, 256>(a, s);
    return bwd<DT, 1, 0, 1024>(a, s);
}

}  // namespace

hipError_t launch_norm_fwd(const NormArgs &a0, hipStream_t s) {
    NormArgs a = a0;
    const int64_t most = 1 << 21, es = a.dtype == LSMX_F32 ? 4 : 2;   // a launch has fewer than 2^32 threads
    for (int64_t at = 0; at < a0.rows; at += most) {
        a.rows = a0.rows - at < most ? a0.rows - at : most;
        auto row = [&](const void *p, int64_t bytes) { return p ? (uint8_t *)p + at * bytes : nullptr; };
        a.x = row(a0.x, a.ldx * es), a.r = row(a0.r, a.ldr * es);
        a.h = row(a0.h, a.dim * es), a.y = row(a0.y, a.dim * es);
        a.codes = row(a0.codes, a.dim), a.scale = row(a0.scale, a.dim / 32);
        const hipError_t e = a.dtype == LSMX_F32 ? fwd_of<LSMX_F32>(a, s) : a.dtype == LSMX_BF16 ? fwd_of<LSMX_BF16>(a, s) : fwd_of<LSMX_F16>(a, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// Workgroups of the backward pass: four a CU, each with a share of dw.
int norm_bwd_groups(int64_t rows) { return (int)(rows < 1024 ? rows : 1024); }

hipError_t launch_norm_bwd(const NormBwdArgs &a, hipStream_t s) {
    hipError_t e = a.dtype == LSMX_F32 ? bwd_of<LSMX_F32>(a, s) : a.dtype == LSMX_BF16 ? bwd_of<LSMX_BF16>(a, s) : bwd_of<LSMX_F16>(a, s);
    if (e != hipSuccess || !a.dw) return e;
    const int groups = norm_bwd_groups(a.rows);
    const unsigned grid = (unsigned)((a.dim + 15) / 16);
    if (a.w_dtype == LSMX_F32)
        norm_dw_kernel<LSMX_F32><<<grid, 1024, 0, s>>>(a.part, groups, a.dim, a.dw);
    else if (a.w_dtype == LSMX_BF16)
        norm_dw_kernel<LSMX_BF16><<<grid, 1024, 0, s>>>(a.part, groups, a.dim, a.dw);
    else
        norm_dw_kernel<LSMX_F16><<<grid, 1024, 0, s>>>(a.part, groups, a.dim, a.dw);
    return hipGetLastError();
}

}  // namespace lsmx
