// dc_act.hip -- 8-bit checkpoints of activations: an activation function whose input is kept in 8 bits for the backward
// pass, in one pass over the data, and the backward pass from that checkpoint.
//
// 32 consecutive values (in the logical order of the rows x cols array) share a power-of-two step 2^k, the smallest with
// amax <= 127.5 * 2^k and k >= -126, and are kept as whole numbers of steps,
//     code = clamp(rint(x / 2^k), -127, 127),   x^ = code 2^k,   |x - x^| <= 2^(k-1):
// scaling by a power of two is exact, so the codes are those of exact arithmetic and x^ is exact in bfloat16 and f32 (f16:
// down to its smallest values).  A value that is not finite is kept as -128 and comes back as NaN.  The checkpoint is the
// codes (32 bytes per group, the last group padded with zeros), then a byte k + 126 per group.
//
// A lane takes 8 consecutive values, so the 4 lanes of a DPP quad hold a group.  All of it is bound by HBM where the
// arrays are large: each byte is moved once, in 16-byte pieces.  (16384 x 8192, bf16: gelu with its checkpoint 102 us, the
// checkpoint back as floats 65, 5.6 TB/s; silu's gated backward pass with its output, 8192 x 8192, 110 us, 6.1 TB/s; a copy
// reaches 5.9.  Arrays of 0.1 to 0.3 million values: 3 to 4 us, a launch.)
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "dc_shared.h"
#include "../../include/dc_gpu.h"

namespace {

using dc::ActArgs;

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f8 __attribute__((ext_vector_type(8)));

static __device__ __forceinline__ float asf(uint32_t u) { return __uint_as_float(u); }
static __device__ __forceinline__ uint32_t asu(float f) { return __float_as_uint(f); }

template <int DT> struct Elem;
template <> struct Elem<DC_F32> { typedef float T; typedef f8 V; static constexpr float MOST = 3.402823466e38f; };
template <> struct Elem<DC_F16> { typedef _Float16 T; typedef h8 V; static constexpr float MOST = 65504.0f; };
template <> struct Elem<DC_BF16> { typedef __bf16 T; typedef b8 V; static constexpr float MOST = 3.38953139e38f; };

// 1 / x and e^x by the hardware's instructions; WIDE (f32 results): with the rounding error of the exponent's argument
static __device__ __forceinline__ float over(float x) { return __builtin_amdgcn_rcpf(x); }
template <bool WIDE> static __device__ __forceinline__ float exp_of(float x, float k = 0.0f) {  // e^x 2^k
    const float hi = x * 1.44269504088896340736f, e = __builtin_amdgcn_exp2f(hi + k);           // (k is not 0 where |hi| > k alone: an exact sum)
    if constexpr (!WIDE) return e;
    const float lo = fmaf(x, 1.44269504088896340736f, -hi) + x * 1.925963033500e-8f;
    return fabsf(lo) < 1.0f ? fmaf(e, lo * 0.69314718055994530942f, e) : e;                     // (x infinite: lo is NaN)
}

// silu: f = x sigma, f' = sigma (1 + x (1 - sigma)).  f32: from e^-|x|, in units of 2^-64 where it is small, so that the tail
// keeps its precision down to the smallest normal result and no power overflows; 16 bits: from e^-x, whose reciprocal is 0
// below -87 (results of less than 2^-119).
// gelu: f = x Phi(x), f' = Phi(x) + x phi(x).  With t = 1 / (1 + c |x|) the upper tail is Phi(-|x|) = e^(-x^2/2) t p(t), p a
// polynomial fitted to it, for f32 of degree 8 (relative error below 6e-8 for every x), for 16 bits of degree 5 (8e-6: the
// forward pass is bound by its arithmetic, not by HBM, with the longer one).  Both by iterated weighted least squares, as
// tests/test_act_fit.py does again.
template <int KIND, bool WIDE> static __device__ __forceinline__ void value_slope(float x, float& f, float& df) {
    if constexpr (KIND == DC_ACT_SILU && WIDE) {
        const float a = fabsf(x), unit = a > 64.0f ? 5.421010862427522e-20f : 1.0f;
        const float e = exp_of<true>(-a, a > 64.0f ? 64.0f : 0.0f), s = over(fmaf(e, unit, 1.0f)), r = e * s, small = r * unit;
        f = x < 0.0f ? x * r * unit : x * s;
        df = fmaf(f, x < 0.0f ? s : small, x < 0.0f ? small : s);
    } else if constexpr (KIND == DC_ACT_SILU) {
        const float e = exp_of<false>(-x), s = over(1.0f + e);
        f = x * s;
        df = fmaf(f, 1.0f - s, s);                          // (x sigma (1 - sigma): finite wherever f is)
    } else {
        const float a = fabsf(x);
        float t, p, e;
        if constexpr (WIDE) {
            t = over(fmaf(a, 0.35355339059327376f, 1.0f));
            p = -0.02969324142f;
            p = fmaf(p, t, 0.1430620308f);
            p = fmaf(p, t, -0.2452032745f);
            p = fmaf(p, t, 0.1408667302f);
            p = fmaf(p, t, -0.01457431771f);
            p = fmaf(p, t, 0.1018762813f);
            p = fmaf(p, t, 0.1214175596f);
            p = fmaf(p, t, 0.1412060496f);
            p = fmaf(p, t, 0.1410421657f);
            e = exp_of<true>(-0.5f * x * x);
        } else {
            t = over(fmaf(a, 0.30935921676911454f, 1.0f));
            p = -0.0724743027f;
            p = fmaf(p, t, 0.177926669f);
            p = fmaf(p, t, 0.0188289209f);
            p = fmaf(p, t, 0.131555132f);
            p = fmaf(p, t, 0.120597981f);
            p = fmaf(p, t, 0.123569132f);
            e = __builtin_amdgcn_exp2f(x * (x * -0.72134752044448170368f));
        }
        const float q = p * t * e, phi = x < 0.0f ? q : 1.0f - q;
        f = x * phi;
        df = fmaf(x, e * 0.39894228040143267794f, phi);
    }
}

// ---- 8 values of a lane -----------------------------------------------------------------------------------------------
// MODE 0: the arrays are flat (rows behind one another) and 16-byte aligned; MODE 1: rows apart, cols and strides whole
// multiples of 8 values; MODE 2: anything, value by value
template <int MODE> struct Place {
    long long i, row, col;              // the lane's first value
    int n;                              // how many of the 8 there are
    __device__ __forceinline__ Place(const ActArgs& a) {
        i = ((long long)blockIdx.x * 256 + threadIdx.x) * 8;
        const long long left = a.n - i;
        n = left < 0 ? 0 : left > 8 ? 8 : (int)left;
        row = col = 0;
        if constexpr (MODE == 1) {
            const uint32_t chunk = (uint32_t)(i >> 3), r = a.cols8_inv ? (uint32_t)__umul64hi(chunk, a.cols8_inv) : chunk;
            row = r;
            col = (long long)(chunk - r * (uint32_t)(a.cols >> 3)) * 8;
        } else if constexpr (MODE == 2) {
            row = i / a.cols;
            col = i - row * a.cols;
        }
    }
};
template <int DT, int MODE> static __device__ __forceinline__ f8 load8(const ActArgs& a, const Place<MODE>& p, const void* x, long long ld) {
    typedef typename Elem<DT>::T T;
    typedef typename Elem<DT>::V V;
    f8 f = {0, 0, 0, 0, 0, 0, 0, 0};
    const T* s = (const T*)x + (MODE == 0 ? p.i : p.row * ld + p.col);
    if (MODE == 2 || p.n < 8) {
        long long row = p.row, col = p.col;
        for (int j = 0; j < p.n; j++) {
            f[j] = (float)(MODE == 0 ? s[j] : ((const T*)x)[row * ld + col]);
            if (MODE != 0 && ++col == a.cols) { col = 0; row++; }
        }
    } else f = __builtin_convertvector(*(const V*)s, f8);
    return f;
}
template <bool PAST, class V> static __device__ __forceinline__ void put(V* p, V x) {
    if constexpr (PAST) __builtin_nontemporal_store(x, p);
    else *p = x;
}
template <int DT, int MODE, bool PAST> static __device__ __forceinline__ void store8(const ActArgs& a, const Place<MODE>& p, void* x, long long ld, f8 f) {
    typedef typename Elem<DT>::T T;
    typedef typename Elem<DT>::V V;
    T* d = (T*)x + (MODE == 0 ? p.i : p.row * ld + p.col);
    if (MODE == 2 || p.n < 8) {
        long long row = p.row, col = p.col;
        for (int j = 0; j < p.n; j++) {
            (MODE == 0 ? d[j] : ((T*)x)[row * ld + col]) = (T)f[j];
            if (MODE != 0 && ++col == a.cols) { col = 0; row++; }
        }
    } else put<PAST>((V*)d, __builtin_convertvector(f, V));
}

template <int CTRL> static __device__ __forceinline__ uint32_t quad(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
}
// the lane's 8 codes and, from the quad's first lane, the group's step (lanes behind the last value take part with zeros)
static __device__ __forceinline__ void keep8(const ActArgs& a, long long i, f8 x, uint8_t* kept) {
    float top = 0.0f;                                       // (NaN if a value is)
#pragma unroll
    for (int j = 0; j < 8; j++) top = __builtin_elementwise_maximum(top, fabsf(x[j]));
    const bool odd = !(top < INFINITY);
    if (odd) {
        top = 0.0f;
        for (int j = 0; j < 8; j++) top = fabsf(x[j]) < INFINITY ? fmaxf(top, fabsf(x[j])) : top;
    }
    uint32_t big = asu(top);
    big = max(big, quad<0xB1>(big));
    big = max(big, quad<0x4E>(big));
    // 127.5 = 255/256 * 2^7: k = exponent - 6, one more where the significand is above 255/128
    int k = (int)(big >> 23) - 127 - 6 + ((big & 0x7FFFFFu) > 0x7F0000u ? 1 : 0);
    k = max(k, -126);
    const float down = asf((uint32_t)(127 - k) << 23);
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        uint32_t c[4];
#pragma unroll
        for (int j = 0; j < 4; j++)                         // 1.5 * 2^23 added: rounded, and the code in the low byte
            c[j] = asu(__builtin_amdgcn_fmed3f(fmaf(x[4 * h + j], down, 12582912.0f), 12582912.0f - 127.0f, 12582912.0f + 127.0f));
        w[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x00000400u), __builtin_amdgcn_perm(c[1], c[0], 0x00000400u), 0x05040100u);
    }
    if (odd) {
        for (int j = 0; j < 8; j++)
            if (!(fabsf(x[j]) < INFINITY)) w[j >> 2] = (w[j >> 2] & ~(0xFFu << (8 * (j & 3)))) | 0x80u << (8 * (j & 3));
    }
    if (i < a.groups * 32) {
        *(uint2*)(kept + i) = make_uint2(w[0], w[1]);
        if ((threadIdx.x & 3) == 0) kept[a.groups * 32 + (i >> 5)] = (uint8_t)(k + 126);
    }
}
// the lane's 8 values back (0 behind the last group)
static __device__ __forceinline__ f8 back8(const ActArgs& a, long long i, const uint8_t* kept) {
    f8 x = {0, 0, 0, 0, 0, 0, 0, 0};
    if (i >= a.groups * 32) return x;
    const uint2 c = *(const uint2*)(kept + i);
    const uint32_t e = kept[a.groups * 32 + (i >> 5)];
    const float s = asf(min(max(e + 1u, 1u), 254u) << 23);  // 2^(e - 126)
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = (float)(int8_t)(w[j >> 2] >> (8 * (j & 3))) * s;
    // seldom: NaNs (a byte 0x80) and the largest steps, whose multiples may pass the largest number
    const uint32_t z0 = w[0] ^ 0x80808080u, z1 = w[1] ^ 0x80808080u;
    const uint32_t nan = ((z0 - 0x01010101u) & ~z0 & 0x80808080u) | ((z1 - 0x01010101u) & ~z1 & 0x80808080u);
    if (nan || e >= 247u)
        for (int j = 0; j < 8; j++)
            x[j] = (int8_t)(w[j >> 2] >> (8 * (j & 3))) == -128 ? asf(0x7FC00000u) : fminf(fmaxf(x[j], -3.402823466e38f), 3.402823466e38f);
    return x;
}

// PAST: the outputs pass the caches (the checkpoint does not: written so in 8-byte pieces it costs 118 us instead of 101).
// KIND 0: the checkpoint alone
template <int DT, int KIND, bool GATED, int MODE, bool PAST> __global__ __launch_bounds__(256) void act_forward(ActArgs a) {
    const Place<MODE> p(a);
    const f8 x = load8<DT, MODE>(a, p, a.x, a.ldx);
    f8 u;
    if constexpr (GATED) u = load8<DT, MODE>(a, p, a.up, a.ldup);
    if constexpr (KIND != DC_ACT_NONE) {
        f8 y;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float f, df;
            value_slope<KIND, DT == DC_F32>(x[j], f, df);
            if constexpr (GATED) f *= u[j];
            y[j] = f;
        }
        store8<DT, MODE, PAST>(a, p, a.y, a.ldy, y);
    }
    keep8(a, p.i, x, a.kept);
    if constexpr (GATED) keep8(a, p.i, u, a.kept_up);
}

// KIND 0: the values read back
template <int DT, int KIND, bool GATED, int MODE, bool PAST> __global__ __launch_bounds__(256) void act_backward(ActArgs a) {
    const Place<MODE> p(a);
    f8 x = back8(a, p.i, a.kept);
    if constexpr (KIND == DC_ACT_NONE) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = x[j] != x[j] ? x[j] : fminf(fmaxf(x[j], -Elem<DT>::MOST), Elem<DT>::MOST);
        store8<DT, MODE, PAST>(a, p, a.dx, a.lddx, x);
    } else {
        const f8 dy = load8<DT, MODE>(a, p, a.x, a.ldx);
        f8 u, dx, du, y;
        if constexpr (GATED) u = back8(a, p.i, a.kept_up);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float f, df;
            value_slope<KIND, DT == DC_F32>(x[j], f, df);
            if constexpr (GATED) {
                dx[j] = dy[j] * u[j] * df;
                du[j] = dy[j] * f;
                y[j] = f * u[j];
            } else {
                dx[j] = dy[j] * df;
                y[j] = f;
            }
        }
        store8<DT, MODE, PAST>(a, p, a.dx, a.lddx, dx);
        if constexpr (GATED) store8<DT, MODE, PAST>(a, p, a.dup, a.lddup, du);
        if (a.y) store8<DT, MODE, PAST>(a, p, a.y, a.ldy, y);
    }
}

template <int DT, int KIND, bool GATED> int go(const ActArgs& a, bool back, hipStream_t st) {
    const unsigned grid = (unsigned)((a.n + 2047) / 2048);
#define DC_MODE(M, P) \
    case 2 * M + P: \
        if (back) act_backward<DT, KIND, GATED, M, P><<<grid, 256, 0, st>>>(a); \
        else act_forward<DT, KIND, GATED, M, P><<<grid, 256, 0, st>>>(a); \
        break
    switch (2 * a.mode + (a.mode < 2 && a.past)) {
        DC_MODE(0, false);
        DC_MODE(0, true);
        DC_MODE(1, false);
        DC_MODE(1, true);
        DC_MODE(2, false);
    }
#undef DC_MODE
    return hipGetLastError() != hipSuccess;
}
template <int DT> int go_kind(const ActArgs& a, bool back, hipStream_t st) {
    if (a.kind == DC_ACT_NONE) return go<DT, DC_ACT_NONE, false>(a, back, st);
    if (a.kind == DC_ACT_SILU) return a.gated ? go<DT, DC_ACT_SILU, true>(a, back, st) : go<DT, DC_ACT_SILU, false>(a, back, st);
    return a.gated ? go<DT, DC_ACT_GELU, true>(a, back, st) : go<DT, DC_ACT_GELU, false>(a, back, st);
}

}  // namespace

extern "C" int dc_launch_act(const dc::ActArgs* a, int back, dc_hip_stream st) {
    if (a->dtype == DC_F32) return go_kind<DC_F32>(*a, back, st);
    if (a->dtype == DC_F16) return go_kind<DC_F16>(*a, back, st);
    return go_kind<DC_BF16>(*a, back, st);
}
