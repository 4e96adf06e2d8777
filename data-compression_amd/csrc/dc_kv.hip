// dc_kv.hip -- a key/value cache held in 4 or 8 bits: quantised as it is written, read back, and attended to as it is
// held (no float copy of it in HBM).
//
// A row is the D keys (or values) of one token and one head.  With n = 2^BITS - 1 it is stored as D codes and one word,
// its step s (a bfloat16, low half) and its zero point z (int16, high half):
//     x^_i = s (z + code_i),   |x_i - x^_i| <= s / 2 (up to f32's rounding of the row's span),
//     s = the smallest bfloat16 >= max(span / n, amax / 32512, 2^-100),  z = rint(lo / s),
//     code_i = clamp(rint(x_i / s) - z, 0, n)           (rint: to nearest, ties to even, of the exact quotient).
// s (z + code) has at most 8 + 15 significant bits, so it is exact in f32 and the only rounding on the way back is the
// one to the output's type.  A row with a value that is not finite has s = NaN and reads back as NaN.
//
// A page holds P tokens (a multiple of 16) of every head; per head: the keys' codes [token][D], the values' codes
// [block of 16 tokens][16 units of D/16 values][16 tokens], the keys' words [token], the values' words [token].  Both
// code layouts put what one lane of the attention's matrix instructions needs into consecutive bytes, so that a wave
// reads a block of 16 tokens of either as one contiguous piece.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <utility>
#include "dc_shared.h"
#include "../../include/dc_gpu.h"

namespace {

using dc::KvArgs;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

static __device__ __forceinline__ float asf(uint32_t u) { return __uint_as_float(u); }
static __device__ __forceinline__ uint32_t asu(float f) { return __float_as_uint(f); }

// ---- element types ------------------------------------------------------------------------------------------------
struct F32 {
    typedef float T;
    static __device__ __forceinline__ float to(T x) { return x; }
    static __device__ __forceinline__ T from(float x) { return x; }
    static constexpr float MOST = 3.402823466e38f;
};
struct F16 {
    typedef _Float16 T;
    static __device__ __forceinline__ float to(T x) { return (float)x; }
    static __device__ __forceinline__ T from(float x) { return (_Float16)x; }
    static constexpr float MOST = 65504.0f;
};
struct BF16 {
    typedef uint16_t T;
    static __device__ __forceinline__ float to(T x) { return asf((uint32_t)x << 16); }
    static __device__ __forceinline__ T from(float x) {                 // to nearest, ties to even
        const __bf16 y = (__bf16)x;
        return __builtin_bit_cast(uint16_t, y);
    }
    static constexpr float MOST = 3.38953139e38f;
};

// N values at p, moved in pieces of A bytes (what the alignment allows)
template <class T, int N, int A> static __device__ __forceinline__ void load_n(const T* p, T* x) {
    constexpr int BYTES = N * (int)sizeof(T);
    if constexpr (A >= 16 && BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; i++) ((uint4*)x)[i] = ((const uint4*)p)[i];
    } else if constexpr (A >= 8 && BYTES % 8 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 8; i++) ((uint2*)x)[i] = ((const uint2*)p)[i];
    } else if constexpr (A >= 4 && BYTES % 4 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 4; i++) ((uint32_t*)x)[i] = ((const uint32_t*)p)[i];
    } else if constexpr (A >= 2 && BYTES % 2 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 2; i++) ((uint16_t*)x)[i] = ((const uint16_t*)p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < BYTES; i++) ((uint8_t*)x)[i] = ((const uint8_t*)p)[i];
    }
}
template <class T, int N, int A> static __device__ __forceinline__ void store_n(T* p, const T* x) {
    constexpr int BYTES = N * (int)sizeof(T);
    if constexpr (A >= 16 && BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; i++) ((uint4*)p)[i] = ((const uint4*)x)[i];
    } else if constexpr (A >= 8 && BYTES % 8 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 8; i++) ((uint2*)p)[i] = ((const uint2*)x)[i];
    } else if constexpr (A >= 4 && BYTES % 4 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 4; i++) ((uint32_t*)p)[i] = ((const uint32_t*)x)[i];
    } else if constexpr (A >= 2 && BYTES % 2 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 2; i++) ((uint16_t*)p)[i] = ((const uint16_t*)x)[i];
    } else {
#pragma unroll
        for (int i = 0; i < BYTES; i++) ((uint8_t*)p)[i] = ((const uint8_t*)x)[i];
    }
}

// the same past the caches, 16 bytes at a time
template <class T, int N> static __device__ __forceinline__ void load_past(const T* p, T* x) {
    static_assert(N * (int)sizeof(T) % 16 == 0, "whole pieces");
#pragma unroll
    for (int i = 0; i < N * (int)sizeof(T) / 16; i++) ((u4*)x)[i] = __builtin_nontemporal_load((const u4*)p + i);
}
template <class T, int N> static __device__ __forceinline__ void store_past(T* p, const T* x) {
    static_assert(N * (int)sizeof(T) % 16 == 0, "whole pieces");
#pragma unroll
    for (int i = 0; i < N * (int)sizeof(T) / 16; i++) __builtin_nontemporal_store(((const u4*)x)[i], (u4*)p + i);
}

// n / d by the host's reciprocal m = floor(2^64 / d) + 1 (d = 1: m = 0): exact for n d < 2^64
static __device__ __forceinline__ uint32_t div_by(uint32_t n, unsigned long long m) {
    return m ? (uint32_t)__umul64hi((unsigned long long)n, m) : n;
}

// lane T of the row's 16
template <int T> static __device__ __forceinline__ uint32_t row_lane(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x150 + T, 0xF, 0xF, true);
}
template <int T> static __device__ __forceinline__ float row_lane(float x) { return asf(row_lane<T>(asu(x))); }
template <int... I, class F> static __device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F f) {
    (f(std::integral_constant<int, I>{}), ...);
}

// rotations within a DPP row
template <int N> static __device__ __forceinline__ float ror16(float x) {
    return asf((uint32_t)__builtin_amdgcn_update_dpp(0, (int)asu(x), 0x120 + N, 0xF, 0xF, false));
}
// (these minima and maxima are NaN if a value is)
static __device__ __forceinline__ float least(float a, float b) { return __builtin_elementwise_minimum(a, b); }
static __device__ __forceinline__ float most(float a, float b) { return __builtin_elementwise_maximum(a, b); }
static __device__ __forceinline__ float min16(float x) {
    x = least(x, ror16<8>(x)); x = least(x, ror16<4>(x)); x = least(x, ror16<2>(x)); return least(x, ror16<1>(x));
}
static __device__ __forceinline__ float max16(float x) {
    x = most(x, ror16<8>(x)); x = most(x, ror16<4>(x)); x = most(x, ror16<2>(x)); return most(x, ror16<1>(x));
}

// the smallest bfloat16 c >= 2^-100 with c * n >= v and c * m >= w, from estimates of v / n and w / m that are not above
// them and at most two bfloat16s below (the products are exact: 8 + 8 bits)
static __device__ __forceinline__ float step_up(float v, float inv_n, float n, float w, float inv_m, float m) {
    float c = asf(asu(fmaxf(fmaxf(v * inv_n, w * inv_m) * 0.9999990f, 7.888609052210118e-31f)) & 0xFFFF0000u);
#pragma unroll
    for (int i = 0; i < 2; i++) c = (c * n < v || c * m < w) ? asf(asu(c) + 0x10000u) : c;
    return c;
}

// 1.5 * 2^23 + rint(x / s) of the exact quotient (|x / s| < 2^15), the whole number in the low bits.  The quotient is put
// right by its remainder, which is exact (s has 8 bits), and rounded as x / s itself would be but for 2^-22 of a unit.  That
// is half between two whole numbers only if x / s is: these can be told to a bit, and any other x / s is further from one
// than half a unit, by 2^-8 of it or more (x - s (k + 1/2) is a multiple of x's unit or of half of s's).
static __device__ __forceinline__ uint32_t rint_div(float x, float s, float inv) {
    const float q = x * inv;
    return asu(fmaf(fmaf(-q, s, x), inv, q) + 12582912.0f);
}

// ---- write and read ----------------------------------------------------------------------------------------------------
// A wave takes the up to 16 tokens of one block of the cache, for a head: their keys or their values to write them (its
// arithmetic bounds the write: more, shorter waves), both to read them (the loads' latency bounds the read).  Lane (u, g) =
// (lane % 16, lane / 16) has the unit u (D/16 values) of the tokens 4 g .. 4 g + 3.  A token's values are then 16 lanes'
// consecutive pieces, its smallest and largest value are found within a DPP row, and four tokens' codes of a unit are
// consecutive bytes of the values' layout.  All loads of a wave are on their way before the first is used.
//
// Write: 3 prompts of 4095 tokens, 8 heads of 128, f16 to 4 bits, 17 us, 3.7 TB/s; its vector instructions (8 for a value's
// code, 3 for its row's span) are 10 us of it, before which its loads and behind which its stores are waited for.  64 single
// tokens: 3.8 us.  Read: 4 histories of up to 16384, bf16, 47 us, 5.8 TB/s, what a copy reaches; 3 prompts 12 us.
struct Block {
    uint32_t b, h;
    int t0, n;                          // t0: the call's token at the block's first place (may be negative)
    int kv;                             // write: keys or values
    const uint8_t* base;                // the head's bytes in the page; null: not in the cache
    uint32_t at;                        // the block's first place in the page
};
typedef __attribute__((address_space(4))) int Const;    // lengths, tables: no kernel writes them, so scalar loads will do

template <bool WRITE> static __device__ __forceinline__ bool block_of(const KvArgs& a, Block& k) {
    long long w = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (w >= a.rows) return false;
    k.kv = WRITE ? (int)(w & 1) : 0;
    if (WRITE) w >>= 1;
    const uint32_t x = (uint32_t)w, y = div_by(x, a.heads_inv);
    k.h = x - y * a.heads;
    k.b = div_by(y, a.tokens_inv);                          // (the inverse of the blocks per sequence)
    const int blk = (int)(y - k.b * a.blocks), first = ((const Const*)a.start)[k.b];
    k.n = a.lens ? min(max(((const Const*)a.lens)[k.b], 0), a.tokens) : a.tokens;
    const long long p0 = (long long)(first & ~15) + 16ll * blk;
    k.t0 = 16 * blk - (first & 15);
    k.base = nullptr;
    k.at = 0;
    if (p0 >= 0 && p0 < a.capacity) {
        const uint32_t slot = div_by((uint32_t)p0, a.page_inv);
        k.at = (uint32_t)p0 - slot * a.page;
        const int page = a.table ? ((const Const*)a.table)[(long long)k.b * a.table_stride + slot] : (int)k.b;
        if (page >= 0 && page < a.pages) k.base = a.data + ((long long)page * a.heads + k.h) * a.head_bytes;
    }
    return true;
}

// PAST: the input passes the caches
template <class E, int D, int BITS, bool VEC, bool PAST> __global__ __launch_bounds__(256) void kv_write(KvArgs a) {
    constexpr int N = D / 16, U = N * BITS / 8, ROW = 16 * U;
    constexpr int BYTES = N * (int)sizeof(typename E::T);
    constexpr int AL = VEC ? (BYTES & -BYTES) : (int)sizeof(typename E::T);
    constexpr int CODES = (1 << BITS) - 1;
    Block k;
    if (!block_of<true>(a, k)) return;
    const int u = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3, t = k.t0 + 4 * g;
    bool on[4], all = true, any = false;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        on[r] = t + r >= 0 && t + r < k.n;
        all &= on[r];
        any |= on[r];
    }
    if (!k.base) {
        if (any && u == 0) atomicOr(a.status, 1u);
        return;
    }
    const typename E::T* src = (k.kv ? (const typename E::T*)a.v + k.b * a.vs[0] + k.h * a.vs[2]
                                     : (const typename E::T*)a.k + k.b * a.ks[0] + k.h * a.ks[2]) + u * N;
    const long long stride = k.kv ? a.vs[1] : a.ks[1];
    alignas(16) typename E::T raw[4][N];
    if (!all) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int i = 0; i < N; i++) raw[r][i] = E::from(0.0f);
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (on[r]) {
            if constexpr (PAST && VEC && BYTES % 16 == 0) load_past<typename E::T, N>(src + (t + r) * stride, raw[r]);
            else load_n<typename E::T, N, AL>(src + (t + r) * stride, raw[r]);
        }
    // the four rows' smallest and largest values; then their steps and zero points, row u % 4 by lane u for all
    float x[4][N], lo[4], hi[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        lo[r] = hi[r] = 0.0f;
        if (!__any(on[r])) continue;                        // (single tokens: one of the four)
#pragma unroll
        for (int i = 0; i < N; i++) x[r][i] = E::to(raw[r][i]);
        lo[r] = hi[r] = x[r][0];
#pragma unroll
        for (int i = 1; i < N; i++) {
            lo[r] = least(lo[r], x[r][i]);
            hi[r] = most(hi[r], x[r][i]);
        }
        lo[r] = min16(lo[r]);
        hi[r] = max16(hi[r]);
    }
    const int own = u & 3;
    const float l = own & 2 ? (own & 1 ? lo[3] : lo[2]) : own & 1 ? lo[1] : lo[0];
    const float h = own & 2 ? (own & 1 ? hi[3] : hi[2]) : own & 1 ? hi[1] : hi[0];
    const float s = step_up(0.5f * h - 0.5f * l, 2.0f / (float)CODES, 0.5f * (float)CODES, fmaxf(h, -l), 1.0f / 32512.0f, 32512.0f);
    const float inv = __builtin_amdgcn_rcpf(s);
    const uint32_t z = rint_div(l, s, inv);
    const bool finite = most(fabsf(l), fabsf(h)) < INFINITY;
    const uint32_t word = finite ? (asu(s) >> 16) | z << 16 : 0x7FC0u;     // (else a step of NaN, codes of 0)
    const uint32_t top = finite ? CODES : 0;
    uint8_t* codes = (uint8_t*)k.base + (k.kv ? (long long)a.page * ROW : 0) + (long long)k.at * ROW;
    uint32_t* words = (uint32_t*)((uint8_t*)k.base + 2ll * a.page * ROW + (k.kv ? 4ll * a.page : 0)) + k.at + 4 * g;
    if (u < 4 && t + u >= 0 && t + u < k.n) words[u] = word;
    alignas(16) uint8_t out[4][U];
    each_of(std::make_integer_sequence<int, 4>{}, [&](auto I) {
        constexpr int r = I.value;
        if (!__any(on[r])) return;
        const float sr = row_lane<r>(s), ir = row_lane<r>(inv);
        // added as its negative: x less a lane's whole number becomes v_subrev_u32 with DPP, which moves the other
        // operand instead (of any control, measured; sums, minima and the f32 forms move the one that is named)
        const uint32_t zr = row_lane<r>(0u - z), most = row_lane<r>(top);
#pragma unroll
        for (int i = 0; i < N; i += 8 / BITS) {
            uint32_t q = 0;
#pragma unroll
            for (int j = 0; j < 8 / BITS; j++)
                q |= (uint32_t)min(max((int)(rint_div(x[r][i + j], sr, ir) + zr), 0), (int)most) << (j * BITS);
            out[r][i * BITS / 8] = (uint8_t)q;
        }
        if (!all && on[r])
            store_n<uint8_t, U, (U & -U)>(codes + (k.kv ? u * (16 * U) + (4 * g + r) * U : (4 * g + r) * ROW + u * U), out[r]);
    });
    if (all) {
        if (k.kv) store_n<uint8_t, 4 * U, (4 * U & -(4 * U))>(codes + u * (16 * U) + g * (4 * U), out[0]);
        else
#pragma unroll
            for (int r = 0; r < 4; r++) store_n<uint8_t, U, (U & -U)>(codes + (4 * g + r) * ROW + u * U, out[r]);
    }
}

// PAST: the output passes the caches
template <class E, int D, int BITS, bool VEC, bool PAST> __global__ __launch_bounds__(256) void kv_read(KvArgs a) {
    constexpr int N = D / 16, U = N * BITS / 8, ROW = 16 * U;
    constexpr int BYTES = N * (int)sizeof(typename E::T);
    constexpr int AL = VEC ? (BYTES & -BYTES) : (int)sizeof(typename E::T);
    Block k;
    if (!block_of<false>(a, k)) return;
    const int u = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3, t = k.t0 + 4 * g, end = a.zero_padding ? a.tokens : k.n;
    if (k.t0 >= end) return;
    typename E::T* dst[2] = {(typename E::T*)a.k + k.b * a.ks[0] + k.h * a.ks[2] + u * N,
                             (typename E::T*)a.v + k.b * a.vs[0] + k.h * a.vs[2] + u * N};
    alignas(16) uint8_t in[2][4][U];
    alignas(16) uint32_t word[2][4];
    if (k.base) {
        const uint8_t* codes = k.base + (long long)k.at * ROW;
        const uint8_t* words = k.base + 2ll * a.page * ROW + 4ll * (k.at + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; r++) load_n<uint8_t, U, (U & -U)>(codes + (4 * g + r) * ROW + u * U, in[0][r]);
        load_n<uint8_t, 4 * U, (4 * U & -(4 * U))>(codes + (long long)a.page * ROW + u * (16 * U) + g * (4 * U), in[1][0]);
        *(uint4*)word[0] = *(const uint4*)words;
        *(uint4*)word[1] = *(const uint4*)(words + 4ll * a.page);
    } else {
        if (t + 3 >= 0 && t < k.n && u == 0) atomicOr(a.status, 1u);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            word[i >> 2][i & 3] = 0x7FC0u;                  // NaN
            for (int j = 0; j < U; j++) in[i >> 2][i & 3][j] = 0;
        }
    }
#pragma unroll
    for (int kv = 0; kv < 2; kv++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if (t + r < 0 || t + r >= end) continue;
            const bool pad = t + r >= k.n;
            const float s = pad ? 0.0f : asf(word[kv][r] << 16), z = pad ? 0.0f : (float)((int)word[kv][r] >> 16), zs = s * z;
            const float most = s != s ? s : E::MOST;        // (the median of three NaNs is NaN)
            const bool far = fabsf(zs) > 1e38f;             // s z alone may pass the largest number: in halves
            const float s1 = far ? 0.5f * s : s, zs1 = far ? 0.5f * s * z : zs, twice = far ? 2.0f : 1.0f;
            alignas(16) typename E::T out[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                const uint32_t byte = in[kv][r][i * BITS / 8], code = BITS == 8 ? byte : (i & 1) ? byte >> 4 : byte & 15;
                float x = fmaf((float)code, s1, zs1);       // (s z and s code are exact, and so is their sum)
                x *= twice;
                out[i] = E::from(__builtin_amdgcn_fmed3f(x, -most, most));
            }
            typename E::T* to = dst[kv] + (t + r) * (kv ? a.vs[1] : a.ks[1]);
            if constexpr (PAST && VEC && BYTES % 16 == 0) store_past<typename E::T, N>(to, out);
            else store_n<typename E::T, N, AL>(to, out);
        }
}

// ---- attention ---------------------------------------------------------------------------------------------------------
// O = softmax(scale q k^T) v^ over the positions a query sees.  With k^ = s (z + code):
//     q . k^_t = ks_t q . code_t + ks_t kz_t sum(q),      O_d = sum_t (p_t vs_t) (code_td + vz_t):
// the matrix instructions see the codes alone, as whole numbers (exact), and a token's step and zero point enter as two
// multiply-adds on its score and as a factor of its weight.  The queries of a group of heads that share keys are the
// columns of mfma 16x16x32: A = 16 tokens' codes, B = 16 queries.  The score tile's lane layout (token = 4 (lane / 16) +
// r, query = lane % 16) is that of the weights' operand in the second product if its 32 tokens are taken in the order
// (block of 16, r) for each group of lanes, and the values' layout in the cache has that order: no data crosses lanes.
//
// A code becomes an f16 by its bits alone: in bits 4..7 they are the subnormal code * 2^-20, in bits 0..7 code * 2^-24
// (UNIT), a power of two that is taken out of the sums.  An instruction's sum keeps 24 bits from its largest product's
// exponent on, in which a subnormal counts as 2^-14: it is exact to 2^-18 (4 bits; 2^-14: 8 bits) of a code's unit times the
// largest weight.  (In bits 0..3 that were 2^-14 of 15.)
//
// The weights w_t = p_t vs_t go into the product as f16, in units of each query row's own: p_t is 2 to the power of the score less
// a reference M, and vs_t counts in 2^(R - 7), one power of two for a wave.  M is raised only by what its row sees (`refer`)
// and so that the largest weight yet is 16 or more and below 2^15.  So 11 bits are kept down to 2^-14, fewer below: a weight
// is off by 2^-11 of itself, half a unit of what f16 outputs round to, or by 2^-29 of its row's largest; whatever the steps
// of tokens that a row does not see, or sees with no weight.  (As far as p_t may go: rows whose steps are 2^-80 of the largest
// in their tile lose bits, as do those with scores above 2^20, for which the wave's largest step sets the unit.)  The sum of
// p_t is kept in f32.
// Queries are scaled to 2^14..2^15 by a power of two (exact); elements 2^-30 of a row's largest lose bits.
//
// A token's words are wanted by the 16 lanes that share its 4 tokens of a block: lane % 8 decodes one of the group's 8
// tokens, and the others take the factors from it by DPP (row_newbcast), mostly within the instruction that uses them.
// (Decoded by every lane for itself that was 80 of a step's 300 vector instructions, which bound it at short heads.)
// The scores' sums start from z sum(q), so that one multiplication by ks and one multiply-add to the power of two are left of
// a score's own; with the weights rounded two at a time and the values' operands made by one byte permute for four codes, a
// step of 32 tokens x 32 queries of 64 values is 200 vector instructions (302 before), 16 of them exponentials.
//
// 48 sequences of up to 8192 positions, 8 heads of 128 in 4 bits: 62 us and 4.7 for the join, 4.9 TB/s; bound by HBM, in
// pieces of 2 KiB.  One of 262143, 2 heads: 17.4 + 4.0 us, 4.1 TB/s.  517 positions: 9.0 us, the chain of lengths, pages,
// codes, scores and sums.  Prompts (two of up to 509 queries behind 8192, 16 heads of 64, 8 bits): 63 to 80 us by their
// lengths, 316 to 400 TFLOP/s, 84 % of the vector instructions' rate while the waves run; the longer one's workgroups are
// waited for (cut in pieces they cost their prologues and the join: 72 us, so 72 to 78).
static __device__ __forceinline__ float over_groups_max(float x) {     // over the 4 groups of 16 lanes
    auto p = __builtin_amdgcn_permlane32_swap((int)asu(x), (int)asu(x), false, false);
    x = fmaxf(asf((uint32_t)p[0]), asf((uint32_t)p[1]));
    auto q = __builtin_amdgcn_permlane16_swap((int)asu(x), (int)asu(x), false, false);
    return fmaxf(asf((uint32_t)q[0]), asf((uint32_t)q[1]));
}
static __device__ __forceinline__ float over_groups_sum(float x) {
    auto p = __builtin_amdgcn_permlane32_swap((int)asu(x), (int)asu(x), false, false);
    x = asf((uint32_t)p[0]) + asf((uint32_t)p[1]);
    auto q = __builtin_amdgcn_permlane16_swap((int)asu(x), (int)asu(x), false, false);
    return asf((uint32_t)q[0]) + asf((uint32_t)q[1]);
}

union Frag { h8 v; uint32_t u[4]; };

constexpr float NOTHING = -3.402823466e38f;                 // the reference of a row that has seen nothing: below every score, and finite

template <int BITS> constexpr float UNIT = BITS == 4 ? 1048576.0f : 16777216.0f;
// the codes in both halves of x times 1 / UNIT: 4 bits, four pairs of nibbles 0..3; 8 bits, two of bytes 0..1
template <int BITS> static __device__ __forceinline__ void codes_of(uint32_t x, uint32_t* o) {
    if constexpr (BITS == 4) {
        o[0] = (x << 4) & 0x00F000F0u;
        o[1] = x & 0x00F000F0u;
        o[2] = (x >> 4) & 0x00F000F0u;
        o[3] = (x >> 8) & 0x00F000F0u;
    } else {
        o[0] = x & 0x00FF00FFu;
        o[1] = __builtin_amdgcn_perm(0, x, 0x0C030C01u);
    }
}
// the bytes at offsets oa and ob of w[] (known when this is compiled), one per half
static __device__ __forceinline__ uint32_t byte_pair(const uint32_t* w, int oa, int ob) {
    return __builtin_amdgcn_perm(w[ob / 4], w[oa / 4], (uint32_t)(oa & 3) | 0x0C00u | (uint32_t)((ob & 3) + 4) << 16 | 0x0C000000u);
}

// the d (within 8) that element e of a key operand holds
template <int BITS> static __device__ __forceinline__ constexpr int key_order(int e) {
    if constexpr (BITS == 4) return (e >> 1) + 4 * (e & 1);
    else return (e & 4) + ((e >> 1) & 1) + 2 * (e & 1);
}

template <int U> struct Stage {         // what a lane holds of 32 tokens: 2 blocks of 16
    uint32_t k[2][U], v[2][U];
    uint32_t kw, vw;                    // of token 16 j + 4 g + r, j and r the bits of lane % 8
};
// where a step's two blocks lie: the first byte of their keys' codes and of their words (uniform over a wave), and
// whether they are not in the cache
struct Where {
    const uint8_t *codes[2], *words[2];
    bool hole[2];
};

// a query row's N values from d0 on, and (with the first of them, LSE) the log of its sum
template <int N, bool LSE = true> static __device__ __forceinline__ void put(const KvArgs& a, uint32_t b, uint32_t h, int rw, int d0, const float* o, float lse) {
    const int i = (int)div_by((uint32_t)rw, a.group_inv), hq = (int)h * a.group + rw - i * a.group;
    const long long at = b * a.vs[0] + (long long)i * a.vs[1] + (long long)hq * a.vs[2] + d0;
    if (a.dtype == DC_BF16) {
        alignas(16) uint16_t raw[N];
#pragma unroll
        for (int k = 0; k < N; k++) raw[k] = BF16::from(o[k]);
        if (a.vec_out) store_n<uint16_t, N, (2 * N & -(2 * N))>((uint16_t*)a.v + at, raw);
        else store_n<uint16_t, N, 2>((uint16_t*)a.v + at, raw);
    } else {
        alignas(16) _Float16 raw[N];
#pragma unroll
        for (int k = 0; k < N; k++) raw[k] = (_Float16)o[k];
        if (a.vec_out) store_n<_Float16, N, (2 * N & -(2 * N))>((_Float16*)a.v + at, raw);
        else store_n<_Float16, N, 2>((_Float16*)a.v + at, raw);
    }
    if (LSE && a.lse && d0 == 0) a.lse[((long long)b * a.tokens + i) * a.heads * a.group + hq] = lse;
}
// the log of a row's sum l with the reference m
static __device__ __forceinline__ float log_sum(float m, float l) { return (m + log2f(l)) * 0.69314718055994530942f; }
// 2^(x / 2): the references of waves and pieces may lie so far apart that only the product with what they refer to, taken
// with the root twice, stays in f32's range
static __device__ __forceinline__ float root_exp(float x) { return __builtin_amdgcn_exp2f(0.5f * x); }
// 1 / l; 0 where nothing of what a query sees is in the cache (a token that is has a p of 2^-100 or more), NaN where l is
static __device__ __forceinline__ float inverse_sum(float l) { return l > 0.0f ? 1.0f / l : l; }

// a lane's codes of a block: U words.  PAST (U = 4, an instruction takes whole cache lines): past the caches
template <int U, bool PAST> static __device__ __forceinline__ void load_codes(const uint8_t* p, uint32_t* x) {
    if constexpr (PAST) *(u4*)x = __builtin_nontemporal_load((const u4*)p);
    else load_n<uint32_t, U, 4 * (U & -U)>((const uint32_t*)p, x);
}
template <bool PAST, int U> static __device__ __forceinline__ void load_keys(Stage<U>& c, const Where& at, uint32_t lane_codes) {
#pragma unroll
    for (int j = 0; j < 2; j++) load_codes<U, PAST>(at.codes[j] + lane_codes, c.k[j]);
}
template <bool PAST, int U> static __device__ __forceinline__ void load_values(Stage<U>& c, const Where& at, uint64_t to_values, uint32_t lane_codes) {
#pragma unroll
    for (int j = 0; j < 2; j++) load_codes<U, PAST>(at.codes[j] + to_values + lane_codes, c.v[j]);
}
template <int U> static __device__ __forceinline__ void load_words(Stage<U>& c, const Where& at, uint64_t to_values, bool second, uint32_t lane_words) {
    const uint8_t* p = (second ? at.words[1] : at.words[0]) + lane_words;
    c.kw = *(const uint32_t*)p;
    c.vw = *(const uint32_t*)(p + to_values);
}

// New references for a step whose weights may not fit f16 (or are the first).  `ref` times `unit` are its scores.
//
// R follows the steps where they drift (a largest one below 2^8 R), may pass what f32 holds (above 2^64 R) or scores are so
// large that a reference cannot be moved by single bits; one far above the others is else left to its row's reference, as its
// weights may be nothing.  R does not change what a row's weights are in units of its own: M goes down with 1 / R, as far as L
// then stays below 2^91.  Then M is raised to the row's largest score where that token's weight is still 16 or more, and to
// what makes the largest weight 2^7 .. 2^8 where it would pass 2^15; it is never more than 80 below the largest score, so
// that p and L stay below 2^118.
template <int NT, int N>
static __device__ __forceinline__ void refer(const float (*ref)[8], const float* mx, const float* unit, float vs,
                                             f4 (*acc)[N], float* M, float* L, float* Z, float& R) {
    const float top = over_groups_max(max16(vs >= R ? vs : 0.0f));
    bool far = false;
    float hi[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        hi[nt] = over_groups_max(mx[nt]) * unit[nt];
        far |= fabsf(hi[nt]) > 1048576.0f && fabsf(hi[nt]) < INFINITY;
    }
    int up = 0;                                             // R is raised by 2^up
    if (top >= R && (top < R * 256.0f || top > R * 1.8446744e19f || __any(far))) {
        const uint32_t r = (asu(top) & 0x7F800000u) + 0x00800000u;
        up = (int)(r - asu(R)) >> 23;
        R = asf(r);
    }
    const float vr = vs * asf(0x7F000000u - asu(R)) * 128.0f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float m = M[nt];
        if (up && fabsf(m) < 1048576.0f) m -= (float)min(min(up, 120), max(217 - (int)(asu(over_groups_max(L[nt])) >> 23), 0));
        const float base = fmaxf(m, hi[nt]);
        float x = 0.0f;                                     // the largest weight, with the reference `base`  (NaNs show in the sums)
        each_of(std::make_integer_sequence<int, 8>{}, [&](auto I) {
            constexpr int t = I.value;
            x = fmaxf(x, __builtin_amdgcn_exp2f(fmaf(ref[nt][t], unit[nt], -base)) * row_lane<t>(vr));
        });
        x = over_groups_max(x);
        if (hi[nt] - m > 8.0f && x >= 16.0f) m = hi[nt];
        if (x * __builtin_amdgcn_exp2f(base - m) > 32768.0f) m = base + (float)((int)(asu(x) >> 23) - 134);
        m = fmaxf(m, hi[nt] - 80.0f);
        const float al = M[nt] - m, be = __builtin_amdgcn_exp2f(al - (float)up);
        M[nt] = m;
        L[nt] *= __builtin_amdgcn_exp2f(al);
        Z[nt] *= be;
#pragma unroll
        for (int i = 0; i < N; i++) acc[nt][i] *= be;
    }
}

// One step of a wave: 32 tokens from t0 on against NT tiles of 16 queries.  EDGE: some of them may not be seen.  What the
// registers of `c` held is replaced by the next step's as soon as it is used, so that those loads are under way during the
// rest of this step and the beginning of the next.
template <int D, int BITS, int NT, bool PAST, bool EDGE>
static __device__ __forceinline__ void attend(Stage<D * BITS / 128>& c, const Frag (*q)[D / 32], const float* qsum,
                                              const float* unit, float significand, const int* sees, int t0, int most, int g,
                                              const bool* hole, const Where& next, uint64_t codes_to_values,
                                              uint64_t words_to_values, uint32_t lane_codes, bool second, uint32_t lane_words,
                                              f4 (*acc)[D / 16], float* M, float* L, float* Z, float& R) {
    constexpr int N = D / 16, U = N * BITS / 8, KS = D / 32;
    // the lane's token's words.  (Behind the last position that is seen there may be anything)
    if (EDGE) {
        const int at = t0 + (second ? 16 : 0) + (int)(lane_words >> 2);
        if (at >= most || hole[second]) c.kw = c.vw = 0;
    }
    const float ks = asf(c.kw << 16) * significand, kz = (float)(int16_t)(c.kw >> 16), vs = asf(c.vw << 16), vz = (float)(int16_t)(c.vw >> 16);
    f4 s[NT][2];                                            // from z sum(q) on
    each_of(std::make_integer_sequence<int, 8>{}, [&](auto I) {
        constexpr int t = I.value;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) s[nt][t >> 2][t & 3] = row_lane<t>(kz) * qsum[nt];
    });
#pragma unroll
    for (int st = 0; st < KS; st++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            Frag k;
            codes_of<BITS>(c.k[j][st * BITS / 4], k.u);
            if constexpr (BITS == 8) codes_of<BITS>(c.k[j][2 * st + 1], k.u + 2);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) s[nt][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.v, q[nt][st].v, s[nt][j], 0, 0, 0);
        }
    load_keys<PAST>(c, next, lane_codes);
    float ref[NT][8], mx[NT];                               // (in units of 1 / unit: one multiply-add takes a score to its power)
    int left[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        mx[nt] = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; j++) left[nt][j] = hole[j] ? 0 : sees[nt] - (t0 + 16 * j + 4 * g);   // tokens of this lane that are seen
    }
    each_of(std::make_integer_sequence<int, 8>{}, [&](auto I) {
        constexpr int t = I.value;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float y = s[nt][t >> 2][t & 3] * row_lane<t>(ks);
            if (EDGE && (t & 3) >= left[nt][t >> 2]) y = -INFINITY;
            ref[nt][t] = y;
            mx[nt] = fmaxf(mx[nt], y);
        }
    });
    // a score that passes its row's reference by 8, or a step as large as the unit (not a NaN): new references
    bool raise = vs >= R;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) raise |= fmaf(mx[nt], unit[nt], -M[nt]) > 8.0f;    // (M + 8 is rounded above 2^27)
    if (__any(raise)) refer<NT, N>(ref, mx, unit, vs, acc, M, L, Z, R);
    const float vr = vs * asf(0x7F000000u - asu(R)) * 128.0f;       // 2^7 / R
    Frag w[NT];
    each_of(std::make_integer_sequence<int, 4>{}, [&](auto I) {
        constexpr int t = 2 * I.value;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float p[2], x[2];
#pragma unroll
            for (int k = 0; k < 2; k++) p[k] = __builtin_amdgcn_exp2f(fmaf(ref[nt][t + k], unit[nt], -M[nt]));
            x[0] = p[0] * row_lane<t>(vr);
            x[1] = p[1] * row_lane<t + 1>(vr);
            if (EDGE) {                                     // (0 times a NaN)
#pragma unroll
                for (int k = 0; k < 2; k++)
                    if (((t + k) & 3) >= left[nt][t >> 2]) x[k] = 0.0f;
            }
            asm("" : "+v"(x[0]), "+v"(x[1]));               // (or each weight is rounded twice, for either use)
            uint32_t both = __builtin_bit_cast(uint32_t, (h2){(_Float16)x[0], (_Float16)x[1]});
            asm("" : "+v"(both));
            const h2 wt = __builtin_bit_cast(h2, both);
            L[nt] += p[0] + p[1];
            Z[nt] = fmaf((float)wt[0], row_lane<t>(vz), Z[nt]);
            Z[nt] = fmaf((float)wt[1], row_lane<t + 1>(vz), Z[nt]);
            w[nt].u[t / 2] = both;
        }
    });
    load_words(c, next, words_to_values, second, lane_words);
    // values: unit lane % 16, tokens 4 g .. 4 g + 3 of both blocks; 4 bits: even and odd codes in bits 4..7 of their bytes
    constexpr int ODD = BITS == 4;
    uint32_t v[2][1 + ODD][U];
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
        for (int k = 0; k < U; k++) {
            v[j][0][k] = ODD ? (c.v[j][k] << 4) & 0xF0F0F0F0u : c.v[j][k];
            if (ODD) v[j][ODD][k] = c.v[j][k] & 0xF0F0F0F0u;
        }
#pragma unroll
    for (int i = 0; i < N; i++) {
        Frag f;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int r = 0; r < 2; r++) f.u[2 * j + r] = byte_pair(v[j][i & ODD], 2 * r * U + i * BITS / 8, (2 * r + 1) * U + i * BITS / 8);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) acc[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.v, w[nt].v, acc[nt][i], 0, 0, 0);
    }
    load_values<PAST>(c, next, codes_to_values, lane_codes);
}

static __device__ __forceinline__ int context_of(const KvArgs& a, uint32_t b) {
    return (int)min((long long)max(((const Const*)a.start)[b], 0), a.capacity);
}
// Into how many pieces (at most a.splits) sequence b's positions are cut, and how long they are: all workgroups of a call
// get about the same number of positions, whatever the sequences' lengths, and there are about a.target of them.  (A cut
// by the same number for all takes as long as the longest sequence's piece.)  Called by all lanes of a wave.
static __device__ __forceinline__ int cut(const KvArgs& a, int context, int& pieces) {
    pieces = 1;
    if (a.splits > 1) {
        float total = (float)context;
        if (a.batch > 1) {
            total = 0.0f;
            for (int i = threadIdx.x & 63; i < a.batch; i += 64) total += (float)min((long long)max(a.start[i], 0), a.capacity);
            for (int m = 32; m; m >>= 1) total += __shfl_xor(total, m);
            total = asf(__builtin_amdgcn_readfirstlane(asu(total)));
        }
        const int even = max((int)min(total * (float)a.heads * (float)a.tiles / (float)a.target, 1e9f), 255) + 1;
        pieces = max(min((context + even - 1) / even, (int)a.splits), 1);
    }
    return ((context + pieces - 1) / pieces + 127) & ~127;
}

template <int D, int BITS, int NT, bool PAST> __global__ __launch_bounds__(256) void kv_attention(KvArgs a) {
    constexpr int N = D / 16, U = N * BITS / 8, ROW = 16 * U, KS = D / 32, COLS = 16 * NT;
    constexpr bool ALL = D * NT <= 256;                     // every wave its own sums in LDS, or one after the other
    __shared__ float acc_lds[(ALL ? 4 : 1) * N * 16 * COLS];
    __shared__ float ml[2][4][COLS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    // Workgroup -> (piece, sequence, head, tile of query rows), the tile fastest: workgroups go round the 8 XCDs one by
    // one, and pieces that a short sequence does not have lie together at the end.  (With the piece as the fastest index
    // whole XCDs idle; a head's tiles kept on one XCD are slower where there are few heads, of unequal lengths.)
    uint32_t x = blockIdx.x;
    const uint32_t tile = x % a.tiles; x /= a.tiles;
    const uint32_t h = x % a.heads; x /= a.heads;
    const uint32_t b = x % a.batch, split = x / a.batch;
    const int context = context_of(a, b);
    if (context != ((const Const*)a.start)[b] && threadIdx.x == 0) atomicOr(a.status, 1u);
    const int len = a.lens ? min(max(((const Const*)a.lens)[b], 0), a.tokens) : a.tokens;
    const int rows = len * a.group;
    const int row0 = tile * COLS;
    const int oc = threadIdx.x & 15, ou = threadIdx.x >> 4;     // a thread's output: a row, a unit
    if (a.zero_padding && split == 0) {
        const float zero[N] = {};
        for (int nt = 0; nt < NT; nt++) {
            const int rw = row0 + nt * 16 + oc;
            if (rw >= rows && rw < (int)a.row_slots) put<N, false>(a, b, h, rw, ou * N, zero, 0.0f);
        }
    }
    if (row0 >= rows) return;
    int pieces;
    const int chunk = cut(a, context, pieces);
    if ((int)split >= pieces) return;
    // what the tile's queries see: positions below sees, from least (all of them) to most (the last one)
    const int last_row = min(row0 + COLS, rows) - 1;
    int least = context, most = context;
    if (a.causal) {
        least = max(context - len + 1 + (int)div_by((uint32_t)row0, a.group_inv), 0);
        most = max(context - len + 1 + (int)div_by((uint32_t)last_row, a.group_inv), 0);
    }
    int sees[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int i = (int)div_by((uint32_t)min(row0 + nt * 16 + col, last_row), a.group_inv);
        sees[nt] = a.causal ? max(context - len + 1 + i, 0) : context;
    }
    const long long lo64 = (long long)split * chunk;
    const int lo = lo64 < most ? (int)lo64 : most, hi = (int)min((long long)most, lo64 + chunk);

    // the wave's tokens: 32 of each 128.  Their pages are followed from step to step: a table entry and a block of 16
    // within its page, for the first block and for the one behind it.  (The first ones are loaded before the queries are
    // waited for)
    const Const* table = a.table ? (const Const*)a.table + (long long)b * a.table_stride : nullptr;
    const uint32_t blocks = (uint32_t)a.page >> 4, slot_step = div_by(8u, a.blocks_inv), in_step = 8u - slot_step * blocks;
    const int first = lo + wave * 32;
    uint32_t slot = div_by((uint32_t)first >> 4, a.blocks_inv), in = ((uint32_t)first >> 4) - slot * blocks;
    const uint32_t lane_codes = (uint32_t)(col * ROW + g * (4 * U)), lane_words = (uint32_t)(g * 4 + (lane & 3)) * 4;
    const bool second = lane & 4;
    const uint64_t codes_to_values = (uint64_t)a.page * ROW;
    const uint64_t words_to_values = 4ull * (uint32_t)a.page;
    int page[2];
    uint32_t place[2];
    auto find = [&](int t) {                                // (the second block may lie past the end: then the first again)
        const uint32_t s1 = in + 1 == blocks ? slot + 1 : slot;
        const bool two = t + 16 < hi;
        place[0] = in;
        place[1] = !two ? in : in + 1 == blocks ? 0 : in + 1;
        page[0] = table ? table[slot] : (int)b;
        page[1] = table ? table[two ? s1 : slot] : (int)b;
        in += in_step;
        slot += slot_step;
        if (in >= blocks) { in -= blocks; slot++; }
    };
    auto where = [&](Where& w) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            w.hole[j] = page[j] < 0 || page[j] >= a.pages;
            const uint8_t* base = a.data + ((long long)(w.hole[j] ? 0 : page[j]) * a.heads + h) * a.head_bytes;
            w.codes[j] = base + (uint64_t)place[j] * (16 * ROW);
            w.words[j] = base + 2 * codes_to_values + (uint64_t)place[j] * 64;
        }
    };
    Stage<U> c;
    Where now, next;
    if (first < hi) {
        find(first);
        where(now);
        load_keys<PAST>(c, now, lane_codes);
        load_words(c, now, words_to_values, second, lane_words);
        load_values<PAST>(c, now, codes_to_values, lane_codes);
        if (first + 128 < hi) find(first + 128);
    }

    // queries, as f16 in the keys' order, with the scale's sign; their sum; and the power of two that takes a score to log2
    // units.  (The scale's significand goes with the keys' steps.  A score times its unit is then exact, and its difference
    // from a reference 0 for the score that was made the reference, however large it is)
    const float per_score = fabsf(a.scale) * 1.44269504088896340736f, significand = __builtin_amdgcn_frexp_mantf(per_score);
    const int exponent = __builtin_amdgcn_frexp_expf(per_score) + (BITS == 4 ? 20 : 24);    // (and UNIT's)
    Frag q[NT][KS];
    float qsum[NT], unit[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int rw = min(row0 + nt * 16 + col, last_row);     // (rows behind the last one repeat it; they are not put out)
        const int i = (int)div_by((uint32_t)rw, a.group_inv), gi = rw - i * a.group;
        const long long at = b * a.ks[0] + (long long)i * a.ks[1] + (long long)(h * a.group + gi) * a.ks[2] + g * (D / 4);
        float f[D / 4];
        uint32_t top = 0;
        if (a.dtype == DC_BF16) {
            const uint16_t* p = (const uint16_t*)a.k + at;
            alignas(16) uint16_t raw[D / 4];
            if (a.vec) load_n<uint16_t, D / 4, 16>(p, raw);
            else load_n<uint16_t, D / 4, 2>(p, raw);
#pragma unroll
            for (int j = 0; j < D / 4; j++) f[j] = BF16::to(raw[j]);
        } else {
            const _Float16* p = (const _Float16*)a.k + at;
            alignas(16) _Float16 raw[D / 4];
            if (a.vec) load_n<_Float16, D / 4, 16>(p, raw);
            else load_n<_Float16, D / 4, 2>(p, raw);
#pragma unroll
            for (int j = 0; j < D / 4; j++) f[j] = (float)raw[j];
        }
#pragma unroll
        for (int j = 0; j < D / 4; j++) top = max(top, asu(f[j]) & 0x7FFFFFFFu);
        const float big = over_groups_max(asf(min(top, 0x7F7FFFFFu)));
        const int e = min(268 - (int)(asu(big) >> 23), 253);            // 2^(14 - exponent of the largest)
        const float up = copysignf(asf((uint32_t)e << 23), a.scale), down = asf((uint32_t)(254 - e) << 23);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < KS; j++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const _Float16 v = (_Float16)(f[j * 8 + key_order<BITS>(k)] * up);
                q[nt][j].v[k] = v;
                sum += (float)v;
            }
        qsum[nt] = over_groups_sum(sum) * (1.0f / UNIT<BITS>);
        unit[nt] = fmaxf(__builtin_amdgcn_ldexpf(down, exponent), 1.17549435e-38f);     // (not 0: -inf times it is -inf)
    }

    f4 acc[NT][N];
    float M[NT], L[NT], Z[NT], R = 7.888609052210118e-31f;  // (2^-100: the smallest step)
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        M[nt] = NOTHING;
        L[nt] = Z[nt] = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) acc[nt][i] = (f4){0, 0, 0, 0};
    }

    int t0 = first;
    auto advance = [&] {                                    // (behind the last step its own tokens are loaded once more)
        if (t0 + 128 < hi) {
            where(next);
            if (t0 + 256 < hi) find(t0 + 256);
        }
    };
    // steps whose tokens are all seen, then the others
    while (t0 < hi && t0 + 32 <= least && t0 + 32 <= hi && !now.hole[0] && !now.hole[1]) {
        next = now;
        advance();
        attend<D, BITS, NT, PAST, false>(c, q, qsum, unit, significand, sees, t0, most, g, now.hole, next, codes_to_values, words_to_values,
                                   lane_codes, second, lane_words, acc, M, L, Z, R);
        now = next;
        t0 += 128;
    }
    while (t0 < hi) {
        if ((now.hole[0] || now.hole[1]) && lane == 0) atomicOr(a.status, 1u);
        next = now;
        advance();
        attend<D, BITS, NT, PAST, true>(c, q, qsum, unit, significand, sees, t0, most, g, now.hole, next, codes_to_values, words_to_values,
                                  lane_codes, second, lane_words, acc, M, L, Z, R);
        now = next;
        t0 += 128;
    }

    // the four waves' sums, in a fixed order; each divided by their common sum of weights first, as without that they pass
    // f32's range where values come near to it
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        L[nt] = over_groups_sum(L[nt]);
        Z[nt] = over_groups_sum(Z[nt]);
        if (g == 0) {
            ml[0][wave][nt * 16 + col] = M[nt];
            ml[1][wave][nt * 16 + col] = L[nt];
        }
    }
    __syncthreads();
    auto sums = [&](int c, float& m, float& l) {            // a column's reference and sum of weights
        m = ml[0][0][c];
        l = 0.0f;
        for (int v = 1; v < 4; v++) m = fmaxf(m, ml[0][v][c]);
        for (int v = 0; v < 4; v++) {
            const float sc = root_exp(ml[0][v][c] - m);
            l = fmaf(ml[1][v][c] * sc, sc, l);
        }
    };
    float f[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float m, l;
        sums(nt * 16 + col, m, l);
        f[nt] = root_exp(M[nt] - m) * (R * 0.0078125f) * (root_exp(M[nt] - m) * inverse_sum(l));
    }
    for (int v = 0; v < (ALL ? 1 : 4); v++) {
        if (ALL || wave == v)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        float* p = &acc_lds[(((ALL ? wave : 0) * NT + nt) * N + i) * 256 + (g * 4 + r) * 16 + col];
                        const float y = fmaf(acc[nt][i][r], UNIT<BITS>, Z[nt]) * f[nt];
                        *p = ALL || v == 0 ? y : *p + y;
                    }
        __syncthreads();
    }
    // 16 columns x 16 units: a thread writes the N values of its unit
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int rw = row0 + nt * 16 + oc;
        if (rw >= rows) continue;
        float o[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            float y = 0.0f;
            for (int v = 0; v < (ALL ? 4 : 1); v++) y += acc_lds[((v * NT + nt) * N + i) * 256 + ou * 16 + oc];
            o[i] = y;
        }
        float m = 0.0f, l = 0.0f;
        if (ou == 0) sums(nt * 16 + oc, m, l);
        if (pieces > 1) {                                   // with its reference and sum
            const long long at = ((((long long)b * a.heads + h) * a.row_slots + rw) * a.splits + split);
            float* p = a.part + at * D + ou * N;
            for (int k = 0; k < N; k++) p[k] = o[k];
            if (ou == 0) {
                a.part_ml[2 * at] = m;
                a.part_ml[2 * at + 1] = l;
            }
            continue;
        }
        const bool none = (a.causal ? context - len + 1 + (int)div_by((uint32_t)rw, a.group_inv) : context) <= 0;
        if (none)
            for (int k = 0; k < N; k++) o[k] = 0.0f;
        put<N>(a, b, h, rw, ou * N, o, none ? -INFINITY : log_sum(m, l));
    }
}

// The pieces of a query row joined, in a fixed order.  Few pieces: 32 or 64 lanes for a row, four values each, one piece
// after the other.  (1536 rows of 4 pieces: 4.6 us, of which a launch is 3; so is 16 rows of 256 with the other.)
template <int D> __global__ __launch_bounds__(256) void kv_join_few(KvArgs a) {
    constexpr int LANES = D <= 128 ? 32 : 64, ROWS = 256 / LANES;
    uint32_t x = blockIdx.x;
    const uint32_t row_blocks = (a.row_slots + ROWS - 1) / ROWS;
    const int rw = (int)(x % row_blocks) * ROWS + (int)threadIdx.x / LANES; x /= row_blocks;
    const uint32_t h = x % a.heads, b = x / a.heads;
    const int context = context_of(a, b), len = a.lens ? min(max(((const Const*)a.lens)[b], 0), a.tokens) : a.tokens;
    int pieces;
    cut(a, context, pieces);
    const int d0 = (int)threadIdx.x % LANES * 4;
    if (rw >= len * a.group || pieces == 1 || d0 >= D) return;
    const long long at = (((long long)b * a.heads + h) * a.row_slots + rw) * a.splits;
    float m = NOTHING, l = 0.0f;
    for (int s = 0; s < pieces; s++) m = fmaxf(m, a.part_ml[2 * (at + s)]);
    for (int s = 0; s < pieces; s++) {
        const float f = root_exp(a.part_ml[2 * (at + s)] - m);
        l = fmaf(a.part_ml[2 * (at + s) + 1] * f, f, l);
    }
    const float inv = inverse_sum(l);
    f4 o = {0, 0, 0, 0};
#pragma unroll 4
    for (int s = 0; s < pieces; s++) {
        const float f = root_exp(a.part_ml[2 * (at + s)] - m);
        o += *(const f4*)(a.part + (at + s) * D + d0) * (a.part_ml[2 * (at + s) + 1] * f * f * inv);
    }
    const bool none = (a.causal ? context - len + 1 + (int)div_by((uint32_t)rw, a.group_inv) : context) <= 0;
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; k++) y[k] = none ? 0.0f : o[k];
    put<4>(a, b, h, rw, d0, y, none ? -INFINITY : log_sum(m, l));
}

// Many pieces: a workgroup for 32 values of a row.  The pieces' references and sums first, a thread each (at most 256),
// then 8 x 32 threads, four values of every 32nd piece each.
template <int D> __global__ __launch_bounds__(256) void kv_join(KvArgs a) {
    __shared__ float f[256], red[2][4];
    __shared__ f4 sums[32][8];
    uint32_t x = blockIdx.x;
    const uint32_t d0 = x % (D / 32) * 32; x /= D / 32;
    const uint32_t rw = x % a.row_slots; x /= a.row_slots;
    const uint32_t h = x % a.heads, b = x / a.heads;
    const int context = context_of(a, b), len = a.lens ? min(max(((const Const*)a.lens)[b], 0), a.tokens) : a.tokens;
    int pieces;
    cut(a, context, pieces);
    if ((int)rw >= len * a.group || pieces == 1) return;
    const int tid = threadIdx.x;
    const long long at = (((long long)b * a.heads + h) * a.row_slots + rw) * a.splits;
    float m = NOTHING, l = 0.0f;
    if (tid < pieces) {
        m = a.part_ml[2 * (at + tid)];
        l = a.part_ml[2 * (at + tid) + 1];
    }
    float top = m;
    for (int k = 32; k; k >>= 1) top = fmaxf(top, __shfl_xor(top, k));
    if ((tid & 63) == 0) red[0][tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float scale = root_exp(m - top), own = l * scale * scale;
    l = own;
    for (int k = 32; k; k >>= 1) l += __shfl_xor(l, k);
    if ((tid & 63) == 0) red[1][tid >> 6] = l;
    __syncthreads();
    l = red[1][0] + red[1][1] + red[1][2] + red[1][3];
    f[tid] = own * inverse_sum(l);
    __syncthreads();
    const int dl = tid & 7, sl = tid >> 3;
    f4 o = {0, 0, 0, 0};
    const float* p = a.part + at * D + d0 + dl * 4;
#pragma unroll 4
    for (int s = sl; s < pieces; s += 32) o += *(const f4*)(p + (long long)s * D) * f[s];
    sums[sl][dl] = o;
    __syncthreads();
    if (tid < 32) {
        float y = 0.0f;
        for (int k = 0; k < 32; k++) y += ((const float*)&sums[k][0])[tid];
        const bool none = (a.causal ? context - len + 1 + (int)div_by(rw, a.group_inv) : context) <= 0;
        if (none) y = 0.0f;
        put<1>(a, b, h, (int)rw, (int)d0 + tid, &y, none ? -INFINITY : log_sum(top, l));
    }
}

__global__ void kv_take(unsigned* word) { word[1] = atomicExch(word, 0u); }

template <class E, int BITS, bool VEC> int go_rows(const KvArgs& a, bool write, hipStream_t st) {
    const unsigned grid = (unsigned)((a.rows + 3) / 4);
#define DC_ROWS(D) \
    case D: \
        if (VEC && a.past) { \
            if (write) kv_write<E, D, BITS, VEC, VEC><<<grid, 256, 0, st>>>(a); \
            else kv_read<E, D, BITS, VEC, VEC><<<grid, 256, 0, st>>>(a); \
        } else if (write) kv_write<E, D, BITS, VEC, false><<<grid, 256, 0, st>>>(a); \
        else kv_read<E, D, BITS, VEC, false><<<grid, 256, 0, st>>>(a); \
        break
    switch (a.dim) {
        DC_ROWS(32); DC_ROWS(64); DC_ROWS(96); DC_ROWS(128); DC_ROWS(160); DC_ROWS(192); DC_ROWS(224); DC_ROWS(256);
        default: return 1;
    }
#undef DC_ROWS
    return hipGetLastError() != hipSuccess;
}
template <class E> int go_bits(const KvArgs& a, bool write, hipStream_t st) {
    if (a.bits == 4) return a.vec ? go_rows<E, 4, true>(a, write, st) : go_rows<E, 4, false>(a, write, st);
    return a.vec ? go_rows<E, 8, true>(a, write, st) : go_rows<E, 8, false>(a, write, st);
}

// Tiles of 16 query rows that a wave takes at once where there are more than 16 of them: what leaves two waves per SIMD.
// (509 queries x 16 heads of 64 in 8 bits, two sequences of up to 8192: two tiles 86 us, four 94 with their join; heads of
// 160, 4 bits: two 120, one 154; heads of 192: 64 queries, two 55, one 45.)
constexpr int wide_tiles(int dim) { return dim <= 160 ? 2 : 1; }

template <int D, int BITS> int go_attention(const KvArgs& a, hipStream_t st) {
    const unsigned grid = (unsigned)((long long)a.splits * a.tiles * a.heads * a.batch);
    constexpr int WIDE = wide_tiles(D);
    if constexpr (WIDE > 1) {
        if (a.cols > 16) kv_attention<D, BITS, WIDE, false><<<grid, 256, 0, st>>>(a);
        else if (D * BITS == 512 && a.past) kv_attention<D, BITS, 1, D * BITS == 512><<<grid, 256, 0, st>>>(a);
        else kv_attention<D, BITS, 1, false><<<grid, 256, 0, st>>>(a);
    } else kv_attention<D, BITS, 1, false><<<grid, 256, 0, st>>>(a);
    constexpr int ROWS = D <= 128 ? 8 : 4;                  // (kv_join_few)
    if (a.splits > dc::DC_KV_JOIN_FEW) kv_join<D><<<(unsigned)((long long)a.row_slots * a.heads * a.batch * (D / 32)), 256, 0, st>>>(a);
    else if (a.splits > 1)
        kv_join_few<D><<<(unsigned)((long long)((a.row_slots + ROWS - 1) / ROWS) * a.heads * a.batch), 256, 0, st>>>(a);
    return hipGetLastError() != hipSuccess;
}

}  // namespace

extern "C" int dc_launch_kv_rows(const dc::KvArgs* a, int write, dc_hip_stream st) {
    if (a->dtype == DC_F32) return go_bits<F32>(*a, write, st);
    if (a->dtype == DC_F16) return go_bits<F16>(*a, write, st);
    return go_bits<BF16>(*a, write, st);
}

extern "C" int dc_launch_kv_take(unsigned* word, dc_hip_stream st) {
    kv_take<<<1, 1, 0, st>>>(word);
    return hipGetLastError() != hipSuccess;
}

extern "C" int dc_kv_wide_cols(int dim) { return 16 * wide_tiles(dim); }

extern "C" int dc_launch_kv_attention(const dc::KvArgs* a, dc_hip_stream st) {
#define DC_DIM(D) case D: return a->bits == 4 ? go_attention<D, 4>(*a, st) : go_attention<D, 8>(*a, st)
    switch (a->dim) {
        DC_DIM(32); DC_DIM(64); DC_DIM(96); DC_DIM(128); DC_DIM(160); DC_DIM(192); DC_DIM(224); DC_DIM(256);
        default: return 1;
    }
#undef DC_DIM
}
