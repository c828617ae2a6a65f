// Helpers of the norm, the router and the experts' products: 16- and 32-bit
// elements as fp32, the MXFP8 rule, and the arguments of the launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lsmx_common.h"

namespace lsmx {

// Element types as the kernels are instantiated for them: storage S, and
// conversions.  Rounding to nearest, ties to even.
template <int DT>
struct Elem;
template <>
struct Elem<LSMX_F32> {
    typedef float S;
    static LSMX_DEV float load(S v) { return v; }
    static LSMX_DEV S store(float v) { return v; }
};
template <>
struct Elem<LSMX_BF16> {
    typedef __bf16 S;
    static LSMX_DEV float load(S v) { return (float)v; }
    static LSMX_DEV S store(float v) { return (__bf16)v; }
};
template <>
struct Elem<LSMX_F16> {
    typedef _Float16 S;
    static LSMX_DEV float load(S v) { return (float)v; }
    static LSMX_DEV S store(float v) { return (_Float16)v; }
};

// ------------------------------------------------------------------- MXFP8
// E8M0 byte of a block whose absmax has the fp32 bits `am`: the least power
// of two that keeps the block within 448 = 1.75 * 2^8, so that no element
// saturates.  1 for a block of zeros; NaN for one with an infinity or a NaN.
LSMX_HD uint32_t mx8_byte(uint32_t am) {
    if (am == 0u) return 127u;
    if (am >= 0x7F800000u) return 255u;
    const int e = (int)(am >> 23) - 8 + ((am & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < 0 ? 0u : (uint32_t)e;
}
// 2^(127 - byte), what the block's elements are multiplied by (byte 255: 1)
LSMX_HD float mx8_inverse(uint32_t byte) { return byte == 255u ? 1.f : u2f((254u - byte) << 23); }

// E4M3 codes of a, b, c, d in the bytes of a word (round to nearest even).
LSMX_DEV uint32_t e4m3_x4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Sums of a wave's lanes up to each.
LSMX_DEV int scan64(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast 15, 31
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// --------------------------------------------------------------- arguments
struct NormArgs {
    const void *x, *r, *w;   // r null: no residual
    int dtype, w_dtype;
    int64_t rows, dim, ldx, ldr;
    float eps;
    void *h, *y;             // h null with r null
    uint8_t *codes, *scale;  // null: no MXFP8 form
};
struct NormBwdArgs {
    const void *h, *w, *dy, *dh;  // dh null: no gradient of the sum
    int dtype, w_dtype;
    int64_t rows, dim, ldh, lddy, lddh;
    float eps;
    void *dx, *dw;   // dw null: not wanted
    float *part;     // [norm_bwd_groups, dim]
};
struct RouteArgs {
    const void *logits;
    int dtype;
    int64_t rows, ld;
    int experts, k, sigmoid, groups, top_groups, renorm;
    float scale;
    const float *bias;      // null: none
    const uint8_t *mask;    // null: every row
    float *weights;         // [rows, k]
    int32_t *ids;           // [rows, k]
    const float *dw;        // backward: [rows, k]
    void *dlogits;          // backward: [rows, experts]
};
struct ExpertArgs {
    const uint8_t *x, *xs, *w, *ws;
    const int32_t *ids, *order, *offsets;
    int pairs, k, experts, N, K;
    uint8_t *h, *hs;         // gated: [pairs, N / 2], [pairs, N / 64]
    float *z;                // combine: the pairs' rows, [pairs, ldz]; with zs in
    int64_t ldz;             // fp16 over [pairs, ceil(N / 64)] powers of two
    float *zs;
    const float *weights;
    void *y;
    int y_dtype;
    int64_t tokens;
};

hipError_t launch_norm_fwd(const NormArgs &a, hipStream_t s);
int norm_bwd_groups(int64_t rows);
hipError_t launch_norm_bwd(const NormBwdArgs &a, hipStream_t s);
hipError_t launch_route_fwd(const RouteArgs &a, hipStream_t s);
hipError_t launch_route_bwd(const RouteArgs &a, hipStream_t s);
int64_t dispatch_workspace(int64_t pairs, int experts);
hipError_t launch_dispatch(const int32_t *ids, int pairs, int experts, int32_t *order, int32_t *offsets, int32_t *ws,
                           hipStream_t s);
hipError_t launch_expert_gated(const ExpertArgs &a, hipStream_t s);
hipError_t launch_expert_combine(const ExpertArgs &a, hipStream_t s);

}  // namespace lsmx
