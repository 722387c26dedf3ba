// nkmx.hip — microscaled storage for MI355X (gfx950, CDNA4): 4-bit floating point with its products,
// and 8-bit activation checkpoints with the gradients that read them (include/nkmx.h has the formats).
//
// Two kinds of kernel:
//   * streaming passes (quantize, save, load, gradient of the activation): bound by HBM.  A lane moves 16
//     bytes of numbers per request, a block of 32 columns is 4 or 8 neighbouring lanes, and its largest
//     magnitude travels between them in DPP moves; codes and scales leave in whole contiguous runs;
//   * products: matrix instructions over tiles in LDS.  mx4 operands go to the scaled matrix instruction
//     as they are stored; an 8-bit checkpoint is turned into bf16 on its way into LDS, which is exact
//     (7 bits of magnitude times a power of two).
//
// fp32 arithmetic is IEEE: no fast-math, no contraction, denormals kept.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <tuple>
#include <type_traits>
#include <utility>

#include "nkmx.h"

namespace {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kStep = NKMX_STEP;        // columns of a step
constexpr int kStepBytes4 = kStep / 2;  // its mx4 codes
constexpr uint32_t kInfBits = 0x7F800000u;

// On a lambda: arrays that it captures stay in registers only where it is inlined.
#define NKMX_INLINE __attribute__((always_inline))

// n / d for 32-bit n: one high product with a 64-bit reciprocal (exact: the error of the reciprocal, below
// 2^-64 relative to 1/d, times n < 2^32 stays below 1/d).
struct FastDiv {
    uint64_t inv;  // floor(2^64 / d) + 1, 0 for d = 1
    uint32_t d;
};
inline FastDiv fast_div(uint32_t d) { return FastDiv{d > 1 ? ~0ull / d + 1 : 0, d}; }
__device__ __forceinline__ uint32_t quotient(uint32_t n, FastDiv f)
{
    return f.inv ? (uint32_t)__umul64hi((uint64_t)n, f.inv) : n;
}

// ---------------------------------------------------------------- numbers

template <typename T>
__device__ __forceinline__ float number(T v) { return (float)v; }

// Magnitude bits of an fp32 value: ordered like the magnitudes, infinity and NaN above every number.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// The scale byte of a block from its largest magnitude: the exponent byte of that number less TOP (2 for
// codes up to 6, 6 for codes up to 127), held at 0 = 2^-127; subnormal magnitudes (exponent byte 0) are below
// every scale and get 0 as well.
template <int TOP>
__device__ __forceinline__ uint32_t scale_byte(uint32_t top)
{
    const uint32_t e = top >> 23;
    return e == 255u ? 255u : (e > (uint32_t)TOP ? e - TOP : 0u);
}

// 2^(byte - 127) for bytes below 255 (2^-127 is a subnormal fp32 number); NaN for 255.
__device__ __forceinline__ float scale_value(uint32_t byte)
{
    const uint32_t bits = byte == 0u ? 0x00400000u : byte << 23;
    return __uint_as_float(byte == 255u ? 0x7FC00000u : bits);
}
// 2^(127 - byte) for bytes up to 253 (a finite number's byte is 252 at most).
__device__ __forceinline__ float scale_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// gelu of the 16-bit types.  erfc(|x| / sqrt 2) / 2, the normal distribution's smaller side, by Abramowitz and Stegun's formula
// 7.1.26: erfc(z) = (a1 t + .. + a5 t^5) e^(-z^2), t = 1 / (1 + p z), |error| <= 1.5e-7 (the factors 1 / sqrt 2 and 1 / 2 are in
// the constants).  `tail` gets e^(-x^2 / 2).  Half a step of fp16 is 4.9e-4.
__device__ __forceinline__ float smaller_side(float x, float& tail)
{
    const float u = x * 0.84932180028801905f;  // u^2 = x^2 / (2 ln 2)
    tail = __builtin_amdgcn_exp2f(-(u * u));
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(x), 0.3275911f * 0.70710678118654752f, 1.0f));
    float p = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
    p = fmaf(p, t, 0.5f * 1.421413741f);
    p = fmaf(p, t, 0.5f * -0.284496736f);
    p = fmaf(p, t, 0.5f * 0.254829592f);
    return p * t * tail;
}

// gelu of fp32, to a few roundings of the result.  Up to |x| = 1.25 (Phi(x) - 1/2) / x, and (Phi(x) - 1/2) / x + phi(x) for the
// slope, are polynomials of x^2; beyond, the smaller side is e^(-x^2 / 2) t Q(t) with t = 1 / (1 + |x| / 4), which keeps its
// digits as it vanishes.  The polynomials are least-maximum fits: off by 4e-9 and 1.5e-9 of 1/2, Q by 8e-9 of itself.  Relative
// l2 error over normal inputs 2.8e-8 (slope 3.6e-8), where 0.5 x (1 + erf) in fp32 has 3.9e-8 (4.2e-8) and the formula above
// 8.4e-8 (1.1e-7); 16384 x 4096 takes 93.8 us with it (slope 95.1), 91.6 (89.9) with the formula above.
constexpr float kGeluBorder = 1.25f;
template <int N>
__device__ __forceinline__ float horner(const float (&c)[N], float x)
{
    float r = c[N - 1];
#pragma unroll
    for (int i = N - 2; i >= 0; --i) r = fmaf(r, x, c[i]);
    return r;
}
// t Q(t); `tail` gets e^(-x^2 / 2).
__device__ __forceinline__ float side_over_tail(float x, float& tail)
{
    constexpr float q[] = {0.0997423306f, 0.0995698348f, 0.0952199996f, 0.0711945295f,
                           0.0975557268f, -0.0292390846f, 0.1140797958f, -0.0481649600f};
    tail = __builtin_amdgcn_exp2f((x * x) * -0.72134752044448170f);
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(x), 0.25f, 1.0f));
    return horner(q, t) * t;
}
__device__ __forceinline__ float gelu32(float x)
{
    constexpr float p[] = {0.398942262f, -0.0664899871f, 0.00997150037f, -0.00118270959f, 0.000110327463f, -6.64486106e-6f};
    const float u = x * x, near = fmaf(u, horner(p, u), 0.5f * x);
    float tail;
    const float side = side_over_tail(x, tail);
    const float far = fmaf(-fabsf(x), side * tail, fmaxf(x, 0.0f));
    return fabsf(x) < kGeluBorder ? near : far;
}
__device__ __forceinline__ float gelu32_slope(float x)
{
    constexpr float p[] = {0.797884524f, -0.265961289f, 0.0598397776f, -0.0094937738f, 0.00114656135f, -0.00010654654f, 6.19567072e-6f};
    const float near = fmaf(x, horner(p, x * x), 0.5f);
    float tail;
    const float side = side_over_tail(x, tail);
    const float w = tail * fmaf(fabsf(x), -0.39894228040143268f, side);
    const float far = x < 0.0f ? w : 1.0f - w;
    return fabsf(x) < kGeluBorder ? near : far;
}

__device__ __forceinline__ float logistic(float x)
{
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f));
}

// The logistic function of fp32 in two parts, g + g_low, and 1 - g in two parts, h + h_low.  With e = e^-|x| <= 1 nothing overflows:
// they are 1 / (1 + e) and e / (1 + e), or the other way round.  What the exponential's argument, 1 + e, the reciprocal and
// the product leave behind is carried in the lower parts: in fp32 alone the argument's rounding costs |x| / 2 units of e.  The
// argument stops at 128, where e is 0.
struct Logistic32 {
    float g, g_low, h, h_low;
};
__device__ __forceinline__ Logistic32 logistic32(float x)
{
    const float a = fminf(fabsf(x), 128.0f), high = a * -1.44269502f;  // the upper and the lower part of -1 / ln 2
    const float low = fmaf(a, -1.92596299e-8f, fmaf(a, -1.44269502f, -high));
    const float e = __builtin_amdgcn_exp2f(high), e_low = e * 0.693147182f * low;
    const float d = 1.0f + e, d_low = (e - (d - 1.0f)) + e_low;
    const float q = __builtin_amdgcn_rcpf(d), q_low = fmaf(-q, d_low, fmaf(-q, d, 1.0f)) * q;
    const float p = e * q, p_low = fmaf(e_low, q, fmaf(e, q_low, fmaf(e, q, -p)));
    return x < 0.0f ? Logistic32{p, p_low, q, q_low} : Logistic32{q, q_low, p, p_low};
}
// x g.  Relative l2 error over normal inputs 2.6e-8, from -6 down 3.6e-8 (x / (1 + e^-x) in fp32 3.9e-8 and 3.5e-8, the form of
// the 16-bit types 4.7e-8 and 2.1e-7).  16384 x 4096 91.4 us, as with that form; 1001 x 4097 from the caches 8.7 against 8.1.
__device__ __forceinline__ float silu32(float x)
{
    const Logistic32 l = logistic32(x);
    return fmaf(x, l.g, x * l.g_low);
}
// g (1 + x (1 - g)), 4.4e-8 and 5.9e-8 (4.8e-8 and 5.5e-8; 4.9e-8 and 1.8e-7); 92.3 us against 90.2, 7.8 against 7.1.
__device__ __forceinline__ float silu32_slope(float x)
{
    const Logistic32 l = logistic32(x);
    const float s = fmaf(x, l.h_low, fmaf(x, l.h, 1.0f));
    return fmaf(l.g, s, l.g_low * s);
}

// fn(x) of a number of type T.
template <int FN, typename T>
__device__ __forceinline__ float activation(float x)
{
    if constexpr (FN == NKMX_GELU && std::is_same_v<T, float>) {
        return gelu32(x);
    } else if constexpr (FN == NKMX_GELU) {  // x Phi(x), without a choice by x's sign
        float tail;
        return fmaf(-fabsf(x), smaller_side(x, tail), fmaxf(x, 0.0f));
    } else if constexpr (FN == NKMX_SILU && std::is_same_v<T, float>) {
        return silu32(x);
    } else if constexpr (FN == NKMX_SILU) {
        return x * logistic(x);
    }
    return x;
}
// The same where x may be infinite or NaN: infinity stays, minus infinity times 0 is a NaN.
template <int FN, typename T>
__device__ __forceinline__ float activation_of_any(float x)
{
    const float y = activation<FN, T>(x);
    if ((FN == NKMX_GELU || std::is_same_v<T, float>) && magnitude(x) >= kInfBits) return x > 0.0f ? x : __uint_as_float(0x7FC00000u);
    return y;
}

template <int FN, typename T>
__device__ __forceinline__ float activation_slope(float x)
{
    if constexpr (FN == NKMX_GELU && std::is_same_v<T, float>) {
        return gelu32_slope(x);
    } else if constexpr (FN == NKMX_GELU) {
        float tail;
        const float side = smaller_side(x, tail);
        return fmaf(x * 0.39894228040143268f, tail, x < 0.0f ? side : 1.0f - side);
    } else if constexpr (FN == NKMX_SILU && std::is_same_v<T, float>) {
        return silu32_slope(x);
    } else if constexpr (FN == NKMX_SILU) {
        const float s = logistic(x);
        return s * fmaf(x, 1.0f - s, 1.0f);
    }
    return 1.0f;
}

// ---------------------------------------------------------------- lane exchange

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}
constexpr int kQuadSwap1 = 0xB1, kQuadSwap2 = 0x4E, kHalfMirror = 0x141, kRowRor4 = 0x124, kRowRor8 = 0x128;

// Largest value over the lanes that share a block: 4 lanes of 8 elements or 8 lanes of 4.
template <int LANES>
__device__ __forceinline__ uint32_t block_max(uint32_t v)
{
    v = max(v, dpp<kQuadSwap1>(v));
    v = max(v, dpp<kQuadSwap2>(v));
    if constexpr (LANES == 8) v = max(v, dpp<kHalfMirror>(v));
    return v;
}

// The scale bytes of a DPP row's blocks (4 or 2 of them) side by side, in every lane of the row.
template <int LANES>
__device__ __forceinline__ uint32_t row_scales(uint32_t byte, int lane)
{
    uint32_t v = byte << (8 * ((lane & 15) / LANES));
    if constexpr (LANES == 4) v |= dpp<kRowRor4>(v);
    return v | dpp<kRowRor8>(v);
}

// ---------------------------------------------------------------- memory access

// E neighbouring elements; only the alignment of the type is promised (views start anywhere).
template <typename T, int E>
struct Pack {
    typedef T vec __attribute__((ext_vector_type(E)));
    typedef vec loose __attribute__((aligned(sizeof(T))));
};

template <typename T, int E>
__device__ __forceinline__ typename Pack<T, E>::vec load_pack(const T* p, int64_t live)
{
    typedef typename Pack<T, E>::vec V;
    typedef typename Pack<T, E>::loose L;
    V v;
    if (live >= E) {
        v = __builtin_nontemporal_load(reinterpret_cast<const L*>(p));
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = i < live ? p[i] : (T)0.0f;
    }
    return v;
}

template <typename T, int E>
__device__ __forceinline__ void store_pack(T* p, typename Pack<T, E>::vec v, int64_t live)
{
    typedef typename Pack<T, E>::loose L;
    if (live >= E) {
        __builtin_nontemporal_store(v, reinterpret_cast<L*>(p));
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i < live) p[i] = v[i];
    }
}

template <int BYTES>
struct Word;
template <>
struct Word<2> { typedef uint16_t type; };
template <>
struct Word<4> { typedef uint32_t type; };
template <>
struct Word<8> { typedef u32x2 type; };

// ---------------------------------------------------------------- streaming passes
//
// One lane owns E = 16 bytes / sizeof(T) neighbouring elements; the lanes of a step (128 columns: 16 or 32
// lanes) lie together, and as packed rows have no gaps, lane i of the launch owns codes i * E onwards: codes
// and scales are written (read) as one contiguous run whatever the row length is.  Rows and steps come from
// one division of the step's index.  Workgroups load once, store once and end: the form in which the 2-bit
// quantizer's kernels stream fastest as well.

template <typename T>
struct Lanes {
    static constexpr int E = 16 / (int)sizeof(T);
    static constexpr int step = kStep / E;             // lanes of a step
    static constexpr int block = NKMX_BLOCK / E;       // lanes of a block
    static constexpr int row_blocks = 16 / block;      // blocks of a DPP row
};

// Workgroups of a row of the grid where a launch needs more than one (a constant: the grid's own size would be one more load
// before the first address, 3.9 against 4.0 us for the quantise of 1001 x 4097 fp32).
constexpr uint32_t kGridRow = 1u << 20;

struct Place {
    uint64_t lane;     // index of the lane in the launch
    uint32_t row;
    uint32_t col;
    int64_t live;      // elements of the matrix from this one on, to the end of the row (<= 0 in the padding)
};

// The lane's place number u of U: a wave takes U x 64 neighbouring ones.
template <typename T, int U>
__device__ __forceinline__ bool place_of(Place& p, int u, FastDiv steps, uint32_t n_steps, uint32_t cols)
{
    p.lane = ((uint64_t)blockIdx.y * kGridRow + blockIdx.x) * (256 * U) + (threadIdx.x >> 6) * (64 * U) + u * 64 + (threadIdx.x & 63);
    const uint64_t step = p.lane / Lanes<T>::step;
    if (step >= n_steps) return false;  // all lanes of a step together
    p.row = quotient((uint32_t)step, steps);
    p.col = ((uint32_t)step - p.row * steps.d) * kStep + (uint32_t)(p.lane % Lanes<T>::step) * Lanes<T>::E;
    p.live = (int64_t)cols - (int64_t)p.col;
    return true;
}

template <typename T>
__device__ __forceinline__ void store_scales(uint8_t* scales, const Place& p, uint32_t byte)
{
    const uint32_t v = row_scales<Lanes<T>::block>(byte, (int)(p.lane & 63));
    if ((p.lane & 15) == 0) {
        typedef typename Word<Lanes<T>::row_blocks>::type W;
        reinterpret_cast<W*>(scales)[p.lane / 16] = (W)v;
    }
}

// Largest magnitude of a lane's elements, as fp32 bits.  16-bit types compare two at a time: their magnitude
// bits are ordered as whole numbers too.
__device__ __forceinline__ uint32_t lane_max(Pack<float, 4>::vec v)
{
    return max(max(magnitude(v[0]), magnitude(v[1])), max(magnitude(v[2]), magnitude(v[3])));
}
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t lane_max_halves(u32x4 w)
{
    u16x2 m = __builtin_bit_cast(u16x2, w[0] & 0x7FFF7FFFu);
#pragma unroll
    for (int i = 1; i < 4; ++i)
        m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
    return max((uint32_t)m[0], (uint32_t)m[1]);
}
__device__ __forceinline__ uint32_t lane_max(Pack<bf16, 8>::vec v)
{
    return lane_max_halves(__builtin_bit_cast(u32x4, v)) << 16;
}
__device__ __forceinline__ uint32_t lane_max(Pack<f16, 8>::vec v)
{
    const uint16_t h = (uint16_t)lane_max_halves(__builtin_bit_cast(u32x4, v));
    return __float_as_uint((float)__builtin_bit_cast(f16, h));
}

// mx4 codes of a pair of values, into byte B of `word`.  The convert instruction divides by the scale, rounds
// to the nearest code with ties to even and saturates (checked against the formula for every kind of tie and
// scales from 2^-127 up).
template <int B>
__device__ __forceinline__ uint32_t pair4(uint32_t word, float a, float b, float scale)
{
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, a, b, scale, B);
}
template <int B>
__device__ __forceinline__ uint32_t pair4(uint32_t word, bf16 a, bf16 b, float scale)
{
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, bf16x2{a, b}, scale, B);
}
template <int B>
__device__ __forceinline__ uint32_t pair4(uint32_t word, f16 a, f16 b, float scale)
{
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, f16x2{a, b}, scale, B);
}

template <typename V, int N>
__device__ __forceinline__ uint32_t codes4(V v, float scale)  // N = 4 or 8 values
{
    uint32_t w = pair4<0>(0u, v[0], v[1], scale);
    w = pair4<1>(w, v[2], v[3], scale);
    if constexpr (N == 8) {
        w = pair4<2>(w, v[4], v[5], scale);
        w = pair4<3>(w, v[6], v[7], scale);
    }
    return w;
}

// s + 17/32 bytes an element, as far as memory goes: 16384 x 8192 bf16 (340 MB) 50 .. 52.5 us = 6.5 .. 6.8 TB/s, where
// a large copy runs at 6.9.
template <typename T, int U>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const T* x, uint64_t ldx, uint8_t* codes, uint8_t* scales,
                                                           FastDiv steps, uint32_t n_steps, uint32_t cols)
{
    constexpr int E = Lanes<T>::E;
    Place p[U];
    bool in[U];
    typename Pack<T, E>::vec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        in[u] = place_of<T, U>(p[u], u, steps, n_steps, cols);
        if (in[u]) v[u] = load_pack<T, E>(x + p[u].row * ldx + p[u].col, p[u].live);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (!in[u]) break;
        const uint32_t byte = scale_byte<2>(block_max<Lanes<T>::block>(lane_max(v[u])));
        uint32_t w = codes4<typename Pack<T, E>::vec, E>(v[u], scale_value(byte));
        if (byte == 255u) w = 0u;
        typedef typename Word<E / 2>::type W;
        reinterpret_cast<W*>(codes)[p[u].lane] = (W)w;
        store_scales<T>(scales, p[u], byte);
    }
}

// q = x / 2^e to the nearest whole number: adding 1.5 * 2^23 in one rounding leaves it in the low bits, so
// the byte is cut out of the sum; x * 2^-e is exact inside the fused operation.
__device__ __forceinline__ uint32_t whole8(float x, float inverse)
{
    constexpr float kMagic = 12582912.0f;
    const float s = fmaf(x, inverse, kMagic);
    return __float_as_uint(__builtin_amdgcn_fmed3f(s, kMagic - 127.0f, kMagic + 127.0f));
}

__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    const uint32_t ab = __builtin_amdgcn_perm(b, a, 0x0C0C0400u);
    const uint32_t cd = __builtin_amdgcn_perm(d, c, 0x04000C0Cu);
    return ab | cd;
}

// 2 s + 33/32 bytes an element and, for gelu, some 40 vector instructions: 16384 x 4096 bf16 (338 MB) 54.6 us = 6.2 TB/s
// with both nearly busy; two or four pieces a lane are slower (registers take waves away).
template <typename T, int FN, int U>
__global__ __launch_bounds__(256) void act8_save_kernel(const T* x, uint64_t ldx, T* y, uint64_t ldy, uint8_t* codes,
                                                        uint8_t* scales, FastDiv steps, uint32_t n_steps, uint32_t cols)
{
    constexpr int E = Lanes<T>::E;
    Place p[U];
    bool in[U];
    typename Pack<T, E>::vec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        in[u] = place_of<T, U>(p[u], u, steps, n_steps, cols);
        if (in[u]) v[u] = load_pack<T, E>(x + p[u].row * ldx + p[u].col, p[u].live);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (!in[u]) break;
        const uint32_t byte = scale_byte<6>(block_max<Lanes<T>::block>(lane_max(v[u])));
        const float inverse = scale_inverse(byte == 255u ? 0u : byte);
        uint32_t q[E];
#pragma unroll
        for (int i = 0; i < E; ++i) q[i] = whole8(number(v[u][i]), inverse);
        typedef typename Word<E>::type W;
        W w;
        if constexpr (E == 8) {
            w[0] = low_bytes(q[0], q[1], q[2], q[3]);
            w[1] = low_bytes(q[4], q[5], q[6], q[7]);
            if (byte == 255u) w = W{0u, 0u};
        } else {
            w = low_bytes(q[0], q[1], q[2], q[3]);
            if (byte == 255u) w = 0u;
        }
        if (FN == NKMX_NONE || codes) {
            reinterpret_cast<W*>(codes)[p[u].lane] = w;
            store_scales<T>(scales, p[u], byte);
        }
        if constexpr (FN != NKMX_NONE) {
            typename Pack<T, E>::vec o;
#pragma unroll
            for (int i = 0; i < E; ++i) o[i] = (T)activation<FN, T>(number(v[u][i]));
            if (byte == 255u) {
#pragma unroll
                for (int i = 0; i < E; ++i) o[i] = (T)activation_of_any<FN, T>(number(v[u][i]));
            }
            store_pack<T, E>(y + p[u].row * ldy + p[u].col, o, p[u].live);
        }
    }
}

template <int SEL>
__device__ __forceinline__ void values4(uint32_t w, float scale, float& a, float& b)
{
    const auto v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, SEL);
    a = v[0];
    b = v[1];
}

// The way back: 16384 x 8192 bf16 47 us = 7.2 TB/s.
template <typename T, int U>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(T* out, uint64_t ldo, const uint8_t* codes,
                                                             const uint8_t* scales, FastDiv steps, uint32_t n_steps,
                                                             uint32_t cols)
{
    constexpr int E = Lanes<T>::E;
    typedef typename Word<E / 2>::type W;
    Place p[U];
    bool in[U];
    W code[U];
    uint8_t e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        in[u] = place_of<T, U>(p[u], u, steps, n_steps, cols);
        if (in[u]) {
            code[u] = reinterpret_cast<const W*>(codes)[p[u].lane];
            e[u] = scales[p[u].lane / Lanes<T>::block];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (!in[u]) break;
        const uint32_t w = code[u], byte = e[u];
        const float scale = scale_value(byte == 255u ? 127u : byte);
        float f[8];
        values4<0>(w, scale, f[0], f[1]);
        values4<1>(w, scale, f[2], f[3]);
        if constexpr (E == 8) {
            values4<2>(w, scale, f[4], f[5]);
            values4<3>(w, scale, f[6], f[7]);
        }
        typename Pack<T, E>::vec o;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = (T)(byte == 255u ? __uint_as_float(0x7FC00000u) : f[i]);
        store_pack<T, E>(out + p[u].row * ldo + p[u].col, o, p[u].live);
    }
}

// out = value of the codes (FN none) or dy * fn'(value).  Bytes and bound as in act8_save_kernel: 16384 x 4096 bf16 gelu
// 56 us = 6.0 TB/s.
template <typename T, int FN, int U>
__global__ __launch_bounds__(256) void act8_grad_kernel(T* out, uint64_t ldo, const T* dy, uint64_t ldy,
                                                        const uint8_t* codes, const uint8_t* scales, FastDiv steps,
                                                        uint32_t n_steps, uint32_t cols)
{
    constexpr int E = Lanes<T>::E;
    typedef typename Word<E>::type W;
    Place p[U];
    bool in[U];
    typename Pack<T, E>::vec g[U];
    W code[U];
    uint8_t e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        in[u] = place_of<T, U>(p[u], u, steps, n_steps, cols);
        if (in[u]) {
            code[u] = reinterpret_cast<const W*>(codes)[p[u].lane];
            e[u] = scales[p[u].lane / Lanes<T>::block];
            if constexpr (FN != NKMX_NONE) g[u] = load_pack<T, E>(dy + p[u].row * ldy + p[u].col, p[u].live);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (!in[u]) break;
        const float scale = scale_value(e[u]);
        typename Pack<T, E>::vec o;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            uint32_t four;
            if constexpr (E == 8) four = code[u][i / 4];
            else four = code[u];
            const float v = (float)(int8_t)(four >> (8 * (i & 3))) * scale;
            if constexpr (FN != NKMX_NONE) o[i] = (T)(number(g[u][i]) * activation_slope<FN, T>(v));
            else o[i] = (T)v;
        }
        store_pack<T, E>(out + p[u].row * ldo + p[u].col, o, p[u].live);
    }
}

// The transpose: blocks run down x's columns.  A workgroup of 8 waves takes 256 rows x 64 * CPL columns; a wave
// takes 32 rows = one block of every column, a lane CPL columns (one load of 4 or 8 bytes a row), so a block
// never leaves its lane.  The codes cross LDS once, so that a column's 256 rows leave as 128
// contiguous bytes: whole cache lines.  Bound by memory and by rounds of workgroups that load once and store once, three on a
// CU: 8192 x 4096 fp32 (152 MB, 1024 of them) 26.8 us = 5.7 TB/s.  A further tile column leaves some CUs two in the last round:
// 8192 x 4160 29.1, 8192 x 4224 29.6; with rows off the cache lines, which neighbours then share (5 % more bytes), 8191 x 4097 30.4.
template <typename T, int CPL>
__global__ __launch_bounds__(512) void mx4_quantize_transposed_kernel(const T* x, uint64_t ldx, uint8_t* codes,
                                                                      uint8_t* scales, uint32_t rows, uint32_t cols,
                                                                      uint32_t steps, uint32_t col_tiles)
{
    constexpr int TC = 64 * CPL;
    // 16-byte slots, 8 a column: slot s of column c lies at s ^ (c & 7), so that neither side collides in the banks
    __shared__ u32x4 image[TC * 8];
    __shared__ alignas(16) uint8_t bytes[TC * 8];
    // each XCD takes a contiguous run of tiles: the cache lines that neighbours share are fetched into one L2
    const uint32_t xcd = blockIdx.x & 7u, each = gridDim.x >> 3, more = gridDim.x & 7u;
    const uint32_t t = xcd * each + min(xcd, more) + (blockIdx.x >> 3), tile = t % col_tiles, band = t / col_tiles;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t r0 = band * 256 + wave * 32, c0 = tile * TC + lane * CPL;
    const int live = (int)min((uint32_t)32, rows > r0 ? rows - r0 : 0u);
    const int64_t live_cols = (int64_t)cols - (int64_t)c0;
    typename Pack<T, CPL>::vec v[32];
    const T* p = x + (uint64_t)r0 * ldx + c0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        if (i < live) {
            v[i] = load_pack<T, CPL>(p + (uint64_t)i * ldx, live_cols);
        } else {
#pragma unroll
            for (int j = 0; j < CPL; ++j) v[i][j] = (T)0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) top = max(top, magnitude(number(v[i][j])));
        const uint32_t byte = scale_byte<2>(top);
        const float scale = scale_value(byte);
        u32x4 w;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            uint32_t one = pair4<0>(0u, v[8 * d][j], v[8 * d + 1][j], scale);
            one = pair4<1>(one, v[8 * d + 2][j], v[8 * d + 3][j], scale);
            one = pair4<2>(one, v[8 * d + 4][j], v[8 * d + 5][j], scale);
            one = pair4<3>(one, v[8 * d + 6][j], v[8 * d + 7][j], scale);
            w[d] = byte == 255u ? 0u : one;
        }
        const int c = lane * CPL + j;
        image[c * 8 + (wave ^ (c & 7))] = w;
        bytes[c * 8 + wave] = (uint8_t)byte;
    }
    __syncthreads();
    const uint32_t last = steps * 4;  // blocks of a packed row
    for (int i = threadIdx.x; i < TC * 8; i += 512) {
        const int c = i >> 3, s = i & 7;
        if (tile * TC + c < cols && band * 8 + s < last)
            reinterpret_cast<u32x4*>(codes)[(uint64_t)(tile * TC + c) * last + band * 8 + s] = image[c * 8 + (s ^ (c & 7))];
    }
    for (int i = threadIdx.x; i < TC * 2; i += 512) {  // a step's 4 scale bytes at a time
        const int c = i >> 1, h = i & 1;
        if (tile * TC + c < cols && band * 2 + h < steps)
            reinterpret_cast<uint32_t*>(scales)[(uint64_t)(tile * TC + c) * steps + band * 2 + h] =
                *reinterpret_cast<const uint32_t*>(&bytes[c * 8 + h * 4]);
    }
}

// ---------------------------------------------------------------- mx4 product, few rows
//
// Few rows of a: the call reads b once and is bound by that, and by the look-ups of its scattered lines.  A
// workgroup owns 16 NT rows of b and 16 MT of a; its 8 waves take a run of the steps of k each, straight from memory
// into the operands of the 16 x 16 x 128 instruction (lane l holds row l % 16 and block l / 16 of the step, 16 bytes as
// they are stored: four lanes read 64 bytes of a row, and the next step's load the rest of the cache line), four
// steps at a time, or two, with one load of their scales (16 lines again, for a sixteenth of the bytes).  The waves' sums
// are joined through LDS in wave order.  FUSED: a lane quantizes its own block of 32 numbers of x in registers, with the
// arithmetic of mx4_quantize_kernel.
//
// Rows of a x n x k, codes from HBM: 1 x 4096 x 1024 3.1 us (its 2.2 MB are 0.3): a launch and three memory latencies in a
// chain; 1 x 8192 x 8192 (36 MB) 9.6; 1 x 28672 x 8192 (125 MB) 26.3 = 4.7 TB/s, 1 x 65536 x 4096 (143 MB) 26 = 5.5 TB/s,
// 16 x 28672 x 8192 36: a's rows from L2 are as many bytes as b's then.  Loads of whole lines of 8 rows for two
// instructions each gained nothing over this; k split over 4, 2 or 1 of the waves is slower from k = 4096 on (1 x 8192 x
// 8192 12, 20, 33 us); more waves on a CU by fewer registers too.

constexpr int kRowsWaves = 8;

__device__ __forceinline__ i32x8 operand4(u32x4 v)
{
    return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
}

// The waves' sums of a block of `rows` x `cols` (a power of two) results, in wave order, with the bias, into y.
template <typename T, int SIZE>
__device__ __forceinline__ void join_waves(const float (&sums)[kRowsWaves][SIZE], int cols, T* y, uint64_t ldy, const T* bias,
                                           uint32_t m0, uint32_t n0, uint32_t m, uint32_t n)
{
    for (int i = threadIdx.x; i < SIZE; i += 64 * kRowsWaves) {
        float s = sums[0][i];
#pragma unroll
        for (int w = 1; w < kRowsWaves; ++w) s += sums[w][i];
        const uint32_t row = m0 + i / cols, col = n0 + i % cols;
        if (row < m && col < n) {
            if (bias) s += number(bias[col]);
            y[row * ldy + col] = (T)s;
        }
    }
}

template <typename V>
__device__ __forceinline__ uint32_t eight_max(V v) { return lane_max(v); }
__device__ __forceinline__ uint32_t eight_max(Pack<float, 8>::vec v)
{
    return max(lane_max(Pack<float, 4>::vec{v[0], v[1], v[2], v[3]}), lane_max(Pack<float, 4>::vec{v[4], v[5], v[6], v[7]}));
}

// A block of 32 numbers, `live` of them in the matrix, and its codes as an operand.
template <typename T>
struct Block {
    typename Pack<T, 8>::vec v[4];
    __device__ __forceinline__ void load(const T* p, int64_t live)
    {
        typedef typename Pack<T, 8>::loose L;
        if (live >= 32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const L*>(p + 8 * i);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i / 8][i % 8] = i < live ? p[i] : (T)0.0f;
        }
    }
    __device__ __forceinline__ u32x4 codes(uint32_t& byte) const
    {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, eight_max(v[i]));
        byte = scale_byte<2>(top);
        const float scale = scale_value(byte);
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t one = codes4<typename Pack<T, 8>::vec, 8>(v[i], scale);
            w[i] = byte == 255u ? 0u : one;
        }
        return w;
    }
};

template <typename T, int MT, int NT, bool FUSED>
__global__ __launch_bounds__(64 * kRowsWaves) void mx4_rows_kernel(T* y, uint64_t ldy, const T* x, uint64_t ldx,
                                                                   const uint8_t* ca, const uint8_t* sa, const uint8_t* cb,
                                                                   const uint8_t* sb, const T* bias, uint32_t m, uint32_t n,
                                                                   uint32_t k, uint32_t steps)
{
    __shared__ float sums[kRowsWaves][MT * NT * 256];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const uint32_t col_blocks = (n + 16 * NT - 1) / (16 * NT);
    const uint32_t n0 = blockIdx.x % col_blocks * (16 * NT), m0 = blockIdx.x / col_blocks * (16 * MT);
    const u32x4 *pa[MT], *pb[NT];
    const uint32_t *qa[MT], *qb[NT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const uint64_t row = min(m0 + 16 * t + r, m - 1);
        pa[t] = reinterpret_cast<const u32x4*>(ca) + row * steps * 4 + g;
        qa[t] = reinterpret_cast<const uint32_t*>(sa) + row * steps;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint64_t row = min(n0 + 16 * t + r, n - 1);
        pb[t] = reinterpret_cast<const u32x4*>(cb) + row * steps * 4 + g;
        qb[t] = reinterpret_cast<const uint32_t*>(sb) + row * steps;
    }
    f32x4 acc[MT][NT] = {};
    typedef u32x4 Loose __attribute__((aligned(4)));
    typedef u32x2 Loose2 __attribute__((aligned(4)));
    const auto some = [&](uint32_t s, auto count) NKMX_INLINE {
        constexpr int N = decltype(count)::value;
        u32x4 a[N][MT], b[N][NT], ea[MT], eb[NT];
        const auto scales = [&](const uint32_t* q) NKMX_INLINE {
            if constexpr (N == 4) return *reinterpret_cast<const Loose*>(q + s);
            if constexpr (N == 2) {
                const u32x2 two = *reinterpret_cast<const Loose2*>(q + s);
                return u32x4{two[0], two[1], 0u, 0u};
            }
            return u32x4{q[s], 0u, 0u, 0u};
        };
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            eb[t] = scales(qb[t]);
#pragma unroll
            for (int i = 0; i < N; ++i) b[i][t] = pb[t][(s + i) * 4];
        }
        Block<T> raw[FUSED ? N : 1][FUSED ? MT : 1];
        if constexpr (FUSED) {
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    const uint32_t row = m0 + 16 * t + r, col = (s + i) * kStep + g * 32;
                    if (row < m) raw[i][t].load(x + row * ldx + col, (int64_t)k - (int64_t)col);
                }
        } else {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                ea[t] = scales(qa[t]);
#pragma unroll
                for (int i = 0; i < N; ++i) a[i][t] = pa[t][(s + i) * 4];
            }
            __builtin_amdgcn_sched_barrier(0);  // every load before the first wait: left alone the compiler saves registers
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                uint32_t e;
                if constexpr (FUSED) {
                    a[i][t] = raw[i][t].codes(e);
                    if (m0 + 16 * t + r >= m) {
                        a[i][t] = u32x4{0u, 0u, 0u, 0u};
                        e = 0;
                    }
                } else {
                    e = (ea[t][i] >> (8 * g)) & 255u;
                }
#pragma unroll
                for (int u = 0; u < NT; ++u)
                    acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        operand4(a[i][t]), operand4(b[i][u]), acc[t][u], 4, 4, 0, (int)e, 0, (int)((eb[u][i] >> (8 * g)) & 255u));
            }
    };
    const uint32_t each = (steps + kRowsWaves - 1) / kRowsWaves, end = min(steps, (wave + 1) * each);
    uint32_t s = wave * each;
    for (; s + 4 <= end; s += 4) some(s, std::integral_constant<int, 4>{});
    if (s + 2 <= end) {
        some(s, std::integral_constant<int, 2>{});
        s += 2;
    }
    for (; s < end; ++s) some(s, std::integral_constant<int, 1>{});
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[wave][(16 * t + 4 * g + i) * (16 * NT) + 16 * u + r] = acc[t][u][i];
    __syncthreads();
    join_waves(sums, 16 * NT, y, ldy, bias, m0, n0, m, n);
}

// ---------------------------------------------------------------- tiles

// Workgroup -> tile.  Workgroups go to the 8 XCDs in turn; each XCD takes a contiguous run of tiles, and tiles
// run down bands of 8 tile rows, so that what is resident on one XCD shares operands in its L2.
__device__ __forceinline__ void tile_of(uint32_t b, uint32_t row_tiles, uint32_t col_tiles, uint32_t& tr, uint32_t& tc)
{
    const uint32_t total = row_tiles * col_tiles, xcd = b & 7u, each = total >> 3, more = total & 7u;
    const uint32_t t = xcd * each + min(xcd, more) + (b >> 3);
    const uint32_t band = t / (8 * col_tiles), in = t % (8 * col_tiles);
    const uint32_t high = min(8u, row_tiles - band * 8);
    tr = band * 8 + in % high;
    tc = in / high;
}

// ---------------------------------------------------------------- mx4 product, tiles
//
// A workgroup computes TM x TN of y in waves of WM x WN (32 x 32 x 64 matrix instructions: lane l holds row
// l % 32 and one block of 32 columns).  k goes by in stages of 256 columns = 128 bytes = one cache line a row,
// through two LDS buffers that buffer loads fill directly, one stage ahead.  LDS holds a tile row as 8 slots of
// 16 bytes; slot s of row r lies at s ^ swizzle8(r), so that the 16 rows that are read together do not meet; a
// load writes LDS in lane order, so the lanes' addresses carry the exchange.  The buffer's extent ends the rows: a
// row past the matrix is not read, and its results are not stored.
//
// 8192 x 8192 x 8192: 276 .. 283 us = 3.9 .. 4.0 PFLOP/s in a row of calls, 283 .. 293 between other work; the instructions
// alone would take 139.  The same launch on codes of zeros takes 202: half of what is left is the clock, which falls
// with the power that random operands take.  The rest is LDS, where a wave of 128 x 64 reads 6 operands for 8
// instructions, and the wait at the one barrier of a stage.  Waves of 128 x 128 read a third less and take 267 .. 290 (one a
// SIMD, nothing runs while it waits; 228 on zeros); stages of 64 bytes through four buffers 345 (half lines).

constexpr int kSpan = 4;  // steps whose scales are loaded at a time

// LDS serves 16 lanes' 16 bytes at a time over 256 bytes of banks: of 16 rows at 128 bytes each, those of one
// parity share their banks and need 8 slots of their own.
__device__ __forceinline__ uint32_t swizzle8(uint32_t row) { return (row & 6u) | ((row ^ (row >> 3)) & 1u); }

// The words of a raw buffer's descriptor.
__device__ __forceinline__ u32x4 buffer_of(const void* p, uint32_t bytes)
{
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return u32x4{(uint32_t)a, (uint32_t)(a >> 32) & 0xFFFFu, bytes, 0x00027000u};
}

// 64 lanes load 16 bytes each from `at` of the buffer to LDS from `lds` on, in lane order; what lies past the
// buffer's end is not read (the whole offset is in the lane's register: only that is checked).  Written as
// assembly because the compiler makes every LDS read wait for every such load it knows of, also one into the
// other buffer; nothing comes back in registers.  The caller waits (arrived()) before the barrier that hands
// the data on.  The nop is the wait state between a write of M0 and a load to LDS.
__device__ __forceinline__ void load_to_lds(u32x4 buffer, uint32_t at, const void* lds)
{
    const uint32_t base = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)lds;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :: "s"(base), "v"(at), "s"(buffer) : "memory");
}
// All but the latest LATER loads of every wave have arrived in LDS; what the waves read before is free to be
// overwritten.
template <int LATER = 0>
__device__ __forceinline__ void arrived()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(LATER) : "memory");
}

template <typename T, int TM, int TN, int WM, int WN, int BUFFERS>
__global__ __launch_bounds__(64 * (TM / WM) * (TN / WN)) void mx4_tiles_kernel(
    T* y, uint64_t ldy, const uint8_t* ca, const uint8_t* sa, const uint8_t* cb, const uint8_t* sb, const T* bias,
    uint32_t m, uint32_t n, uint32_t steps, uint32_t row_tiles, uint32_t col_tiles)
{
    constexpr int WAVES = (TM / WM) * (TN / WN), WAVES_N = TN / WN;
    constexpr int FM = WM / 32, FN = WN / 32;
    static_assert(TM % (8 * WAVES) == 0 && TN % (8 * WAVES) == 0 && WAVES % 2 == 0, "whole rounds of row groups");
    __shared__ u32x4 image[BUFFERS][(TM + TN) * 8];
    __shared__ uint32_t bytes[BUFFERS][(TM + (TN < 64 ? 64 : TN)) * kSpan];  // loads of scales are 64 rows long

    uint32_t tr, tc;
    tile_of(blockIdx.x, row_tiles, col_tiles, tr, tc);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, r = lane & 31, g = lane >> 5;
    const int wm = (wave / WAVES_N) * WM, wn = (wave % WAVES_N) * WN;
    const uint32_t stages = (steps + 1) / 2;
    const uint32_t pitch = steps * kStepBytes4, pitch_s = steps * 4;
    const uint32_t rows_a = min((uint32_t)TM, m - tr * TM), rows_b = min((uint32_t)TN, n - tc * TN);
    const u32x4 buf_a = buffer_of(ca + (uint64_t)tr * TM * pitch, rows_a * pitch);
    const u32x4 buf_b = buffer_of(cb + (uint64_t)tc * TN * pitch, rows_b * pitch);
    const u32x4 buf_sa = buffer_of(sa + (uint64_t)tr * TM * pitch_s, rows_a * pitch_s);
    const u32x4 buf_sb = buffer_of(sb + (uint64_t)tc * TN * pitch_s, rows_b * pitch_s);
    // 8 rows a load; a wave's row groups are all even or all odd ones
    const uint32_t at = (lane >> 3) * pitch + (((lane & 7) ^ swizzle8((wave & 1) * 8 + (lane >> 3))) << 4);
    const uint32_t at_s = lane * pitch_s;  // 64 rows a load

    const auto fetch = [&](uint32_t stage) {
        const int buf = stage % BUFFERS;
#pragma unroll
        for (int i = 0; i < TM / 8 / WAVES; ++i) {
            const int group = i * WAVES + wave;
            load_to_lds(buf_a, at + (group * 8 * pitch + stage * 128), &image[buf][group * 64]);
        }
#pragma unroll
        for (int i = 0; i < TN / 8 / WAVES; ++i) {
            const int group = i * WAVES + wave;
            load_to_lds(buf_b, at + (group * 8 * pitch + stage * 128), &image[buf][TM * 8 + group * 64]);
        }
        // Scales of two stages at a time: 16 bytes a row, each in a cache line of its own, whose look-up is what such a
        // load costs
        if ((stage & 1) == 0) {
#pragma unroll
            for (int i = 0; i < (TM / 64 + (TN + 63) / 64 + WAVES - 1) / WAVES; ++i) {
                const int group = i * WAVES + wave;
                uint32_t* to = &bytes[(stage >> 1) % BUFFERS][group * 64 * kSpan];
                if (group < TM / 64)
                    load_to_lds(buf_sa, at_s + (group * 64 * pitch_s + stage * 8), to);
                else if (group < TM / 64 + (TN + 63) / 64)
                    load_to_lds(buf_sb, at_s + ((group - TM / 64) * 64 * pitch_s + stage * 8), to);
            }
        }
    };

    f32x16 acc[FM][FN] = {};
    // Operands of instruction h of a stage: lane g takes block h of the stage's step g (any assignment of blocks
    // to instructions is right as long as both operands agree), so that its four scale bytes are one word that the
    // instructions index themselves.
    struct Operands {
        u32x4 a[FM], b[FN];
    };
    const auto take = [&](Operands& o, int buf, int h) {
        const uint32_t slot = (4 * g + h) ^ swizzle8(r);
#pragma unroll
        for (int j = 0; j < FN; ++j) o.b[j] = image[buf][(TM + wn + 32 * j + r) * 8 + slot];
#pragma unroll
        for (int i = 0; i < FM; ++i) o.a[i] = image[buf][(wm + 32 * i + r) * 8 + slot];
    };
    struct Scales {
        int a[FM], b[FN];
    };
    const auto take_scales = [&](Scales& e, uint32_t stage) {
        const uint32_t* from = bytes[(stage >> 1) % BUFFERS] + (stage & 1) * 2 + g;
#pragma unroll
        for (int i = 0; i < FM; ++i) e.a[i] = from[(wm + 32 * i + r) * kSpan];
#pragma unroll
        for (int j = 0; j < FN; ++j) e.b[j] = from[(TM + wn + 32 * j + r) * kSpan];
    };
    const auto multiply = [&](const Operands& o, const Scales& e, auto index) {
        constexpr int h = decltype(index)::value;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand4(o.a[i]), operand4(o.b[j]), acc[i][j],
                                                                           4, 4, h, e.a[i], h, e.b[j]);
    };
    // While the instructions of one operand set run, the next set is read, a read after every instruction from the
    // first on: left alone the compiler reads late and waits, or reads a whole stage at once, which does not fit
    // the registers.
    const auto interleave = [](auto reads) {
        constexpr int kMfma = 0x008, kLdsRead = 0x100, n = decltype(reads)::value, each = (n + FM * FN - 1) / (FM * FN);
#pragma unroll
        for (int i = 0; i < FM * FN; ++i) {
            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kLdsRead, each, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    typedef std::integral_constant<int, FM + FN> One;
    typedef std::integral_constant<int, 2 * (FM + FN)> Two;

    Operands o, p;
    Scales e, f;
    // Loads of a stage that every wave issues at least; so many of each later stage may be on their way.
    constexpr int LOADS = (TM + TN) / 8 / WAVES;
    const auto one_stage = [&](uint32_t s, const Scales& now, Scales& next, auto more) {
        const int buf = s % BUFFERS;
        if constexpr (decltype(more)::value) fetch(s + BUFFERS - 1);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (FM * FN == 1) {  // one instruction each: what counts is the chain of waits, so everything is read at once
            Operands v, w;
            take(p, buf, 1);
            take(v, buf, 2);
            take(w, buf, 3);
            __builtin_amdgcn_sched_barrier(0);
            multiply(o, now, std::integral_constant<int, 0>{});
            multiply(p, now, std::integral_constant<int, 1>{});
            arrived<decltype(more)::value ? (BUFFERS - 2) * LOADS : 0>();
            take(o, (s + 1) % BUFFERS, 0);
            take_scales(next, s + 1);
            __builtin_amdgcn_sched_barrier(0);
            multiply(v, now, std::integral_constant<int, 2>{});
            multiply(w, now, std::integral_constant<int, 3>{});
            return;
        }
        take(p, buf, 1);
        multiply(o, now, std::integral_constant<int, 0>{});
        interleave(One{});
        take(o, buf, 2);
        multiply(p, now, std::integral_constant<int, 1>{});
        interleave(One{});
        take(p, buf, 3);
        multiply(o, now, std::integral_constant<int, 2>{});
        interleave(One{});
        // this stage has been read; what follows reads the next one while the last instructions run (after the last
        // stage: what is there, unused)
        arrived<decltype(more)::value ? (BUFFERS - 2) * LOADS : 0>();
        take(o, (s + 1) % BUFFERS, 0);
        take_scales(next, s + 1);
        multiply(p, now, std::integral_constant<int, 3>{});
        interleave(Two{});
    };
    const uint32_t whole = steps / 2;
    for (uint32_t s = 0; s + 1 < BUFFERS && s < stages; ++s) fetch(s);
    arrived();
    take(o, 0, 0);
    take_scales(e, 0);
    uint32_t s = 0;
    for (; s + BUFFERS - 1 < stages; ++s) {
        one_stage(s, e, f, std::true_type{});
        e = f;
    }
    for (; s < whole; ++s) {
        one_stage(s, e, f, std::false_type{});
        e = f;
    }
    if (steps & 1) {  // half a stage: the lanes of its second step take part with zeros
        const auto rest = [&](auto index) {
            if (decltype(index)::value) take(o, whole % BUFFERS, decltype(index)::value);
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                if (g) o.a[i] = u32x4{0u, 0u, 0u, 0u};
            }
            multiply(o, e, index);
        };
#pragma unroll
        for (int i = 0; i < FM; ++i) e.a[i] = g ? 0 : e.a[i];
#pragma unroll
        for (int j = 0; j < FN; ++j) e.b[j] = g ? 0 : e.b[j];
        rest(std::integral_constant<int, 0>{});
        rest(std::integral_constant<int, 1>{});
        rest(std::integral_constant<int, 2>{});
        rest(std::integral_constant<int, 3>{});
    }
    arrived();

    // The results cross LDS, 32 rows of the wave at a time, so that they leave in 16-byte pieces of whole lines.
    constexpr int kRowBytes = WN * 4 + 32, E = 16 / (int)sizeof(T), kPerRow = WN / E, kRows = 64 / kPerRow;
    static_assert(WAVES * 32 * kRowBytes <= (int)sizeof(image), "a wave's rows in LDS");
    char* mine = reinterpret_cast<char*>(image) + wave * 32 * kRowBytes;
    const uint32_t col = tc * TN + wn + (lane % kPerRow) * E;
    const int64_t live = (int64_t)n - (int64_t)col;
    float add[E];
#pragma unroll
    for (int c = 0; c < E; ++c) add[c] = bias && c < live ? number(bias[col + c]) : 0.0f;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v)
                *reinterpret_cast<float*>(mine + (8 * (v / 4) + 4 * g + v % 4) * kRowBytes + (32 * j + r) * 4) = acc[i][j][v];
#pragma unroll
        for (int k = 0; k < 32 / kRows; ++k) {
            const int at_row = k * kRows + lane / kPerRow;
            const uint32_t row = tr * TM + wm + 32 * i + at_row;
            const float* from = reinterpret_cast<const float*>(mine + at_row * kRowBytes) + (lane % kPerRow) * E;
            typename Pack<T, E>::vec out;
#pragma unroll
            for (int c = 0; c < E; c += 4) {
                const f32x4 four = *reinterpret_cast<const f32x4*>(from + c);
#pragma unroll
                for (int u = 0; u < 4; ++u) out[c + u] = (T)(bias ? four[u] + add[c + u] : four[u]);
            }
            // cached stores: y is read next, and lines shared with a neighbouring tile meet in L2
            if (row < m) {
                T* to = y + row * ldy + col;
                if (live >= E) {
                    *reinterpret_cast<typename Pack<T, E>::loose*>(to) = out;
                } else {
#pragma unroll
                    for (int c = 0; c < E; ++c)
                        if (c < live) to[c] = out[c];
                }
            }
        }
    }
}

// ---------------------------------------------------------------- weight gradient
//
// dw = dy^T x^: both operands have the contracted index (the token) as their row, so a tile has to be turned
// before the matrix instruction can read it.  A thread loads 8 tokens x 4 columns; packing two tokens of a
// column into one register is also the conversion to bf16 pairs, so the turn is free; a column's 8 tokens go
// to LDS as one 16-byte slot.  x^ = q 2^e has at most 7 bits and is exact in bf16.  dy is cut into PARTS
// bf16 numbers by truncation (1 for bf16, 2 for fp16, 3 for fp32: 8 bits each, exact together), each
// multiplied with x^ in turn: exact products for every type at the bf16 rate, where the fp32 matrix
// instruction has a sixteenth of it.
//
// LDS: column c of a tile is BT tokens = BT / 8 slots; slot s lies at s ^ swizzle_t(c).  t is split over
// blockIdx.y where there are few tiles; the parts are joined in order by a second kernel.
//
// Bound by the matrix instructions and the LDS traffic and turning between them: fp32 16384 x 4352 x 4096 1551 us, 1.13
// PFLOP/s of bf16 products; 5001 x 1023 x 4097 (3 parts of 68 tiles: 204 of 256 CUs) 135 us with the join in a row of calls, 136
// and 12 as single launches.

template <int SLOTS>
__device__ __forceinline__ uint32_t swizzle_t(uint32_t c)
{
    if constexpr (SLOTS == 8) return ((c >> 2) ^ c) & 7u;
    return ((c >> 1) & 2u) | (((c >> 1) ^ (c >> 3)) & 1u);
}

// Two tokens' upper halves side by side (the lower half of the register is the first token).
__device__ __forceinline__ uint32_t upper_halves(uint32_t first, uint32_t second)
{
    return __builtin_amdgcn_perm(second, first, 0x07060302u);
}
__device__ __forceinline__ uint32_t lower_halves(uint32_t first, uint32_t second)
{
    return __builtin_amdgcn_perm(second, first, 0x05040100u);
}

// The upper 8 significant bits of v, and what they leave: an infinity leaves nothing, a NaN a NaN.
__device__ __forceinline__ float upper_part(float v) { return __uint_as_float(__float_as_uint(v) & 0xFFFF0000u); }
__device__ __forceinline__ float rest_of(float v)
{
    return magnitude(v) == kInfBits ? 0.0f : v - upper_part(v);
}

template <typename T>
struct Parts;
template <>
struct Parts<bf16> { static constexpr int count = 1; };
template <>
struct Parts<f16> { static constexpr int count = 2; };
template <>
struct Parts<float> { static constexpr int count = 3; };

// f(0), f(1) .. f(N - 1) with the numbers as constants.
template <typename F, int... I>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>)
{
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F f)
{
    each_of(f, std::make_integer_sequence<int, N>{});
}

// Up to this token every load of a tile stays inside the matrices: a row's end runs on into the next rows, whose
// numbers end in results that are not stored.  `end_d`, `end_x`: the tile's last column + 1 in dy and in the codes.
__device__ __forceinline__ uint32_t safe_tokens(uint32_t t_rows, uint32_t n, uint32_t end_d, uint64_t lddy, uint32_t pitch,
                                                uint32_t end_x)
{
    const uint32_t over_d = end_d > n ? end_d - n : 0, over_x = end_x > pitch ? end_x - pitch : 0;
    const uint32_t ld = (uint32_t)max(lddy, (uint64_t)1);
    const uint32_t rows = max((over_d + ld - 1) / ld, over_x ? (over_x + pitch - 1) / max(pitch, 1u) : 0u);
    return pitch && t_rows > rows ? t_rows - rows : 0;
}

// The scales of a unit's 8 tokens from one scale byte a lane: lane % 8 has that token's, and the 8 lanes around it have
// the same 32 columns.
__device__ __forceinline__ void spread_scales(uint32_t byte, float (&scale)[8])
{
    const int v = __float_as_int(scale_value(byte));
    scale[0] = __int_as_float(__builtin_amdgcn_ds_swizzle(v, 0x18 | 0 << 5));
    scale[1] = __int_as_float(__builtin_amdgcn_ds_swizzle(v, 0x18 | 1 << 5));
    scale[2] = __int_as_float(__builtin_amdgcn_ds_swizzle(v, 0x18 | 2 << 5));
    scale[3] = __int_as_float(__builtin_amdgcn_ds_swizzle(v, 0x18 | 3 << 5));
    scale[4] = __int_as_float(__builtin_amdgcn_ds_swizzle(v, 0x18 | 4 << 5));
    scale[5] = __int_as_float(__builtin_amdgcn_ds_swizzle(v, 0x18 | 5 << 5));
    scale[6] = __int_as_float(__builtin_amdgcn_ds_swizzle(v, 0x18 | 6 << 5));
    scale[7] = __int_as_float(__builtin_amdgcn_ds_swizzle(v, 0x18 | 7 << 5));
}

// Column j of a unit's codes as 8 tokens in bf16.
__device__ __forceinline__ u32x4 eight_tokens(const uint32_t (&q)[8], const float (&scale)[8], int j)
{
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = (float)(int8_t)(q[2 * i] >> (8 * j)) * scale[2 * i];
        const float b = (float)(int8_t)(q[2 * i + 1] >> (8 * j)) * scale[2 * i + 1];
        w[i] = __builtin_bit_cast(uint32_t, bf16x2{(bf16)a, (bf16)b});
    }
    return w;
}

// A wave's part of dw.
template <int FN, int FK>
__device__ __forceinline__ void store_gradient(const f32x16 (&acc)[FN][FK], float* dw, uint64_t lddw, uint32_t row0,
                                               uint32_t col0, uint32_t n, uint32_t k, uint32_t accumulate, int r, int g)
{
#pragma unroll
    for (int j = 0; j < FK; ++j) {
        const uint32_t col = col0 + 32 * j + r;
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const uint32_t row = row0 + 32 * i + 8 * (v / 4) + 4 * g + v % 4;
                if (row < n && col < k) {
                    float* p = dw + row * lddw + col;
                    *p = accumulate ? *p + acc[i][j][v] : acc[i][j][v];
                }
            }
    }
}

template <typename T, int TN, int TK, int WN, int WK, int BT>
__global__ __launch_bounds__(64 * (TN / WN) * (TK / WK)) void act8_wgrad_kernel(
    float* dw, uint64_t lddw, float* db, const T* dy, uint64_t lddy, const uint8_t* codes, const uint8_t* scales,
    uint32_t t_rows, uint32_t n, uint32_t k, uint32_t steps, uint32_t row_tiles, uint32_t col_tiles,
    uint32_t stages_each, uint32_t accumulate, uint64_t part_stride, uint64_t part_stride_db)
{
    constexpr int NT = 64 * (TN / WN) * (TK / WK), WAVES_K = TK / WK, P = Parts<T>::count;
    constexpr int FN = WN / 32, FK = WK / 32, SLOTS = BT / 8, GROUPS = BT / 16;
    constexpr int CD = TN / 4, CX = TK / 4;             // groups of 4 columns
    constexpr int UD = SLOTS * CD, UX = SLOTS * CX;     // units of 8 tokens x 4 columns
    constexpr bool BOTH = UD >= NT;                     // a thread has a unit of each, or one of one
    constexpr int XW = BOTH ? 0 : UD / 64;              // first wave with units of x
    static_assert(BOTH ? (UD == NT && UX == NT) : (UD + UX == NT && UD % 64 == 0), "units and threads");
    __shared__ u32x4 left[2][P][TN * SLOTS];
    __shared__ u32x4 right[2][TK * SLOTS];

    uint32_t tr, tc;
    tile_of(blockIdx.x, row_tiles, col_tiles, tr, tc);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, g = lane >> 5;
    const int wn = (wave / WAVES_K) * WN, wk = (wave % WAVES_K) * WK;
    const uint32_t stages = (t_rows + BT - 1) / BT;
    const uint32_t first = blockIdx.y * stages_each, last = min(stages, first + stages_each);

    // slot (8 tokens) of a unit: the wave's first one and the lane's from there; columns
    const int d_slot0 = wave * 64 / CD, d_slot = d_slot0 + lane / CD, d_col = (lane % CD) * 4;
    const int x_slot0 = (wave - XW) * 64 / CX, x_slot = x_slot0 + lane / CX, x_col = (lane % CX) * 4;
    const uint32_t pitch = steps * kStep, pitch_s = steps * 4, col_x = tc * TK + x_col;
    const uint32_t safe = safe_tokens(t_rows, n, (tr + 1) * TN, lddy, pitch, (tc + 1) * TK);
    typedef std::conditional_t<CD >= 64, uint32_t, uint64_t> At;  // lanes of one row group, or of several rows apart
    const At at_d = (At)(lane / CD) * 8 * (At)lddy * sizeof(T) + d_col * sizeof(T);
    const At at_x = (At)(lane / CX) * 8 * pitch + x_col;
    const At at_s = (At)((lane / CX) * 8 + (lane & 7)) * pitch_s + x_col / 32;

    // Stages up to `safe` load whole tiles; the others element by element, with zeros past the ends.
    typename Pack<T, 4>::vec d[8];
    const auto fetch_d = [&](uint32_t stage) NKMX_INLINE {
        const char* p = reinterpret_cast<const char*>(dy + (uint64_t)(stage * BT + d_slot0 * 8) * lddy + tr * TN);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            d[i] = *reinterpret_cast<const typename Pack<T, 4>::loose*>(p + (uint64_t)i * lddy * sizeof(T) + at_d);
    };
    const auto copy_d = [&](uint32_t stage) NKMX_INLINE {
        const uint32_t t = stage * BT + d_slot * 8;
        const int64_t live = (int64_t)n - (int64_t)(tr * TN + d_col);
        const T* p = dy + (uint64_t)t * lddy + tr * TN + d_col;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                d[i][j] = (T)0.0f;
                if (t + i < t_rows && j < live) d[i][j] = p[(uint64_t)i * lddy + j];
            }
    };
    uint32_t q[8], e;  // codes; scale byte of the unit's token lane % 8
    const auto fetch_x = [&](uint32_t stage) NKMX_INLINE {
        const uint32_t t = stage * BT + x_slot0 * 8;
        const uint8_t* p = codes + (uint64_t)t * pitch + tc * TK;
        e = (scales + (uint64_t)t * pitch_s + tc * (TK / 32))[at_s];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = *reinterpret_cast<const uint32_t*>(p + (uint64_t)i * pitch + at_x);
    };
    const auto copy_x = [&](uint32_t stage) NKMX_INLINE {
        const uint32_t t = stage * BT + x_slot * 8;
        const bool live = col_x < pitch;
        e = 0;
        if (live && t + (lane & 7) < t_rows) e = scales[(uint64_t)(t + (lane & 7)) * pitch_s + col_x / 32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            q[i] = 0u;
            if (live && t + i < t_rows) q[i] = *reinterpret_cast<const uint32_t*>(codes + (uint64_t)(t + i) * pitch + col_x);
        }
    };
    float sum_dy[4] = {};
    // Column j of the unit into LDS.
    const auto put_d = [&](int buf, int j, auto sums) NKMX_INLINE {
        const uint32_t c = d_col + j, at = c * SLOTS + (d_slot ^ swizzle_t<SLOTS>(c));
        if constexpr (P == 1) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a = __builtin_bit_cast(u32x2, d[2 * i])[j / 2];
                const uint32_t b = __builtin_bit_cast(u32x2, d[2 * i + 1])[j / 2];
                const uint32_t two = j % 2 ? upper_halves(a, b) : lower_halves(a, b);
                w[i] = two;
                if constexpr (decltype(sums)::value)
                    sum_dy[j] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, two),
                                                                bf16x2{(bf16)1.0f, (bf16)1.0f}, sum_dy[j], false);
            }
            left[buf][0][at] = w;
        } else {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = number(d[i][j]);
            if constexpr (decltype(sums)::value) {
#pragma unroll
                for (int i = 0; i < 8; ++i) sum_dy[j] += v[i];
            }
#pragma unroll
            for (int part = 0; part < P; ++part) {
                u32x4 w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = upper_halves(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]));
                left[buf][part][at] = w;
                if (part + 1 < P) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = part == 0 ? rest_of(v[i]) : v[i] - upper_part(v[i]);
                }
            }
        }
    };
    float scale[8];
    const auto put_x = [&](int buf, int j) NKMX_INLINE {
        const uint32_t c = x_col + j;
        right[buf][c * SLOTS + (x_slot ^ swizzle_t<SLOTS>(c))] = eight_tokens(q, scale, j);
    };

    f32x16 acc[FN][FK] = {};
    bf16x8 a[FN], b[2][FK];
    const auto take_b = [&](int buf, int h) NKMX_INLINE {
#pragma unroll
        for (int j = 0; j < FK; ++j) {
            const uint32_t c = wk + 32 * j + r;
            b[h & 1][j] = __builtin_bit_cast(bf16x8, right[buf][c * SLOTS + ((2 * h + g) ^ swizzle_t<SLOTS>(c))]);
        }
    };
    const auto take_a = [&](int buf, int u, int i) NKMX_INLINE {  // for step u: 16 tokens u / P, the smallest part first
        const uint32_t c = wn + 32 * i + r;
        a[i] = __builtin_bit_cast(bf16x8, left[buf][P - 1 - u % P][c * SLOTS + ((2 * (u / P) + g) ^ swizzle_t<SLOTS>(c))]);
    };
    // A step: one part of 16 tokens.  An operand is read for the next step as soon as it has been used; those reads and
    // the instructions of what `work` adds go between the matrix instructions.
    constexpr int STEPS = GROUPS * P;
    const auto step = [&](int buf, auto index, auto work) NKMX_INLINE {
        constexpr int u = decltype(index)::value;
        if constexpr (u + 1 < STEPS && (u + 1) % P == 0) take_b(buf, (u + 1) / P);
#pragma unroll
        for (int i = 0; i < FN; ++i) {
#pragma unroll
            for (int j = 0; j < FK; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[(u / P) & 1][j], acc[i][j], 0, 0, 0);
            if constexpr (u + 1 < STEPS) take_a(buf, u + 1, i);
        }
        work();
#pragma unroll
        for (int z = 0; z < FN * FK; ++z) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
            __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);  // others
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // an LDS write
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // A stage; with MORE the next one is loaded at its beginning and turned into the other buffer over its last steps, a
    // column of the units at a time.  D, X: whether this wave has units of dy, of x.
    const auto run = [&](auto sums, auto has_d, auto has_x) NKMX_INLINE {
        constexpr bool D = decltype(has_d)::value, X = decltype(has_x)::value;
        const auto put = [&](int buf, int j) NKMX_INLINE {
            if constexpr (D) put_d(buf, j, sums);
            if constexpr (X) put_x(buf, j);
        };
        const auto stage = [&](uint32_t s, int buf, auto more) NKMX_INLINE {
            constexpr bool MORE = decltype(more)::value;
            if constexpr (MORE) {
                if constexpr (D) fetch_d(s + 1);
                if constexpr (X) fetch_x(s + 1);
            }
            take_b(buf, 0);
#pragma unroll
            for (int i = 0; i < FN; ++i) take_a(buf, 0, i);
            __builtin_amdgcn_sched_barrier(0);
            each<STEPS>([&](auto index) NKMX_INLINE {
                step(buf, index, [&]() NKMX_INLINE {
                    if constexpr (MORE) {
                        constexpr int u = decltype(index)::value, begin = STEPS > 4 ? STEPS - 4 : 1;
                        if (X && u == begin) spread_scales(e, scale);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (min(begin + j, STEPS - 1) == u) put(buf ^ 1, j);
                    }
                });
            });
            __syncthreads();
        };
        const uint32_t fast = max(first, min(last, safe / BT));  // stages of whole tiles
        if (first < fast) {
            if constexpr (D) fetch_d(first);
            if constexpr (X) {
                fetch_x(first);
                spread_scales(e, scale);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) put(0, j);
            __syncthreads();
            int buf = 0;
            for (uint32_t s = first; s + 1 < fast; ++s, buf ^= 1) stage(s, buf, std::true_type{});
            stage(fast - 1, buf, std::false_type{});
        }
#pragma unroll 1
        for (uint32_t s = fast; s < last; ++s) {  // the last tokens
            if constexpr (D) copy_d(s);
            if constexpr (X) {
                copy_x(s);
                spread_scales(e, scale);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) put(0, j);
            __syncthreads();
            stage(s, 0, std::false_type{});
        }
    };
    const auto with_sums = [&](auto has_d, auto has_x) NKMX_INLINE {
        if (db != nullptr && tc == 0) run(std::true_type{}, has_d, has_x);
        else run(std::false_type{}, has_d, has_x);
    };
    if constexpr (BOTH) {
        with_sums(std::true_type{}, std::true_type{});
    } else {  // (both sides meet the same barriers)
        if (wave < XW) with_sums(std::true_type{}, std::false_type{});
        else run(std::false_type{}, std::false_type{}, std::true_type{});
    }

    store_gradient<FN, FK>(acc, dw + blockIdx.y * part_stride, lddw, tr * TN + wn, tc * TK + wk, n, k, accumulate, r, g);
    if (db != nullptr && tc == 0) {  // the token groups' sums of a column, joined in order
        float* part = reinterpret_cast<float*>(&right[0][0]);
        if (BOTH || wave < XW) {
#pragma unroll
            for (int j = 0; j < 4; ++j) part[d_slot * TN + d_col + j] = sum_dy[j];
        }
        __syncthreads();
        if (tid < TN && tr * TN + tid < n) {
            float s = part[tid];
#pragma unroll
            for (int i = 1; i < SLOTS; ++i) s += part[i * TN + tid];
            float* p = db + blockIdx.y * part_stride_db + tr * TN + tid;
            *p = accumulate ? *p + s : s;
        }
    }
}

// The same for bf16 dy on 4-byte boundaries, where nothing has to be cut: dy goes to LDS as it lies in memory, a
// token's columns in a row, by loads that need no registers, and the turn is made by the transposing LDS reads
// (16 lanes read 4 tokens x 16 columns and get 4 tokens of one column each).  A row is TN / 32 pieces of 64 bytes; piece
// c of token t lies at c ^ (t & 3), so that the four tokens that are read together do not meet in the banks.
//
// A stage first asks for the next one's dy and the codes of the one after, then turns the codes that it was given into
// the next stage's operand while its instructions run; the barrier comes before its last 16 tokens, whose
// instructions cover the first reads of the next stage.  Tiles of 64 have one instruction for each 16 tokens and are bound
// by waiting: they read a stage's operands at once and ask for dy three stages ahead (0.62 us a stage against 0.86).
//
// 16384 x 4096 x 4096: 482 us = 1.14 PFLOP/s, where a large bf16 library product runs at 1.20 to 1.35; 16384 x 4096 x 1024 (4
// parts of 64 tiles) 149 us with the join, of which the parts' stores are some 15 and the join 14; with the kernel above 198
// (16384 x 4096 x 4096 673).  On
// zeros both calls take a fifth to an eighth less (390, and 130 with the join): the clock falls with the power of random operands, as for
// the library.  Waves of 64 x 128, late waves, wave priorities, other orders of the tiles and a touch of L2 two stages
// ahead were no faster.
template <int TN, int TK, int WN, int WK>
__global__ __launch_bounds__(64 * (TN / WN) * (TK / WK)) void act8_wgrad_raw_kernel(
    float* dw, uint64_t lddw, float* db, const bf16* dy, uint64_t lddy, const uint8_t* codes, const uint8_t* scales,
    uint32_t t_rows, uint32_t n, uint32_t k, uint32_t steps, uint32_t row_tiles, uint32_t col_tiles,
    uint32_t stages_each, uint32_t accumulate, uint64_t part_stride, uint64_t part_stride_db)
{
    constexpr int WAVES = (TN / WN) * (TK / WK), WAVES_K = TK / WK, BT = 64, SLOTS = BT / 8, GROUPS = BT / 16;
    constexpr int FN = WN / 32, FK = WK / 32, NT = 64 * WAVES;
    constexpr int CX = TK / 4, XWAVES = SLOTS * CX / 64;                // waves with units (8 tokens x 4 columns) of x
    constexpr int PIECES = TN / 32, LR = TN / 8, RP = 64 / LR;          // of a row of dy; lanes of a row, rows of a load
    constexpr int ROWS = BT / WAVES, LOADS = ROWS / RP;                 // rows and loads of a wave
    constexpr int TURN = PIECES < 4 ? PIECES - 1 : 3;
    constexpr bool ALL_X = XWAVES == WAVES;
    constexpr bool SHORT = FN * FK == 1;   // one instruction each: what counts is the chain of waits
    constexpr int DEPTH = SHORT ? 4 : 2;   // buffers of dy
    static_assert(XWAVES <= WAVES && LOADS * RP == ROWS && !(SHORT && ALL_X), "units and waves");
    __shared__ u32x4 left[DEPTH][BT * TN / 8];
    __shared__ u32x4 right[2][TK * SLOTS];

    uint32_t tr, tc;
    tile_of(blockIdx.x, row_tiles, col_tiles, tr, tc);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, g = lane >> 5;
    const int wn = (wave / WAVES_K) * WN, wk = (wave % WAVES_K) * WK;
    const uint32_t stages = (t_rows + BT - 1) / BT;
    const uint32_t first = blockIdx.y * stages_each, last = min(stages, first + stages_each);
    const bool has_x = ALL_X || wave < XWAVES;
    const int x_slot0 = wave * 64 / CX, x_slot = x_slot0 + lane / CX, x_col = (lane % CX) * 4;
    const uint32_t pitch = steps * kStep, pitch_s = steps * 4, col_x = tc * TK + x_col, ld2 = (uint32_t)lddy * 2;
    const uint32_t safe = safe_tokens(t_rows, n, (tr + 1) * TN, lddy, pitch, (tc + 1) * TK);
    typedef std::conditional_t<CX >= 64, uint32_t, uint64_t> At;  // lanes of one row group, or of several rows apart
    const At at_x = (At)(lane / CX) * 8 * pitch + x_col;
    const At at_s = (At)((lane / CX) * 8 + (lane & 7)) * pitch_s + x_col / 32;

    // Stages up to `safe` load whole tiles; the others element by element, with zeros past the ends.
    const auto row_of = [&](int load) NKMX_INLINE { return wave * ROWS + load * RP + lane / LR; };
    const auto fetch_d = [&](uint32_t stage, int buf) NKMX_INLINE {
        const u32x4 from = buffer_of(dy + (uint64_t)(stage * BT) * lddy + tr * TN, (BT - 1) * ld2 + TN * 2);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int p = lane % LR, piece = (p >> 2) ^ (row_of(i) & TURN);
            load_to_lds(from, row_of(i) * ld2 + piece * 64 + (p & 3) * 16, &left[buf][(wave * ROWS + i * RP) * LR]);
        }
    };
    const auto copy_d = [&](uint32_t stage, int buf) NKMX_INLINE {
        uint16_t* to = reinterpret_cast<uint16_t*>(left[buf]);
#pragma unroll 1
        for (int i = tid; i < BT * TN; i += NT) {
            const int t = i / TN, c = i % TN;
            uint16_t v = 0;
            if (stage * BT + t < t_rows && tr * TN + c < n)
                v = reinterpret_cast<const uint16_t*>(dy)[(uint64_t)(stage * BT + t) * lddy + tr * TN + c];
            to[t * TN + ((c >> 5) ^ (t & TURN)) * 32 + (c & 31)] = v;
        }
    };
    struct Unit {
        uint32_t q[8], e;  // codes of 8 tokens x 4 columns; scale byte of token lane % 8 (see the kernel above)
    };
    const auto settle = [&](Unit& u) NKMX_INLINE {
        asm volatile("" : "+v"(u.q[0]), "+v"(u.q[1]), "+v"(u.q[2]), "+v"(u.q[3]), "+v"(u.q[4]), "+v"(u.q[5]), "+v"(u.q[6]),
                     "+v"(u.q[7]), "+v"(u.e));
    };
    const auto fetch_x = [&](Unit& u, uint32_t stage) NKMX_INLINE {
        const uint32_t t = stage * BT + x_slot0 * 8;
        const uint8_t* p = codes + (uint64_t)t * pitch + tc * TK;
        u.e = (scales + (uint64_t)t * pitch_s + tc * (TK / 32))[at_s];
#pragma unroll
        for (int i = 0; i < 8; ++i) u.q[i] = *reinterpret_cast<const uint32_t*>(p + (uint64_t)i * pitch + at_x);
    };
    const auto copy_x = [&](Unit& u, uint32_t stage) NKMX_INLINE {
        const uint32_t t = stage * BT + x_slot * 8;
        const bool live = col_x < pitch;
        u.e = 0;
        if (live && t + (lane & 7) < t_rows) u.e = scales[(uint64_t)(t + (lane & 7)) * pitch_s + col_x / 32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            u.q[i] = 0u;
            if (live && t + i < t_rows) u.q[i] = *reinterpret_cast<const uint32_t*>(codes + (uint64_t)(t + i) * pitch + col_x);
        }
    };
    const auto put_x = [&](const Unit& u, const float (&scale)[8], int buf, int j) NKMX_INLINE {
        const uint32_t c = x_col + j;
        right[buf][c * SLOTS + (x_slot ^ swizzle_t<SLOTS>(c))] = eight_tokens(u.q, scale, j);
    };

    f32x16 acc[FN][FK] = {};
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* LdsShorts;
    // Lane a of 16 reads 4 columns of token a / 4; lanes 0-31 take the first 8 tokens of an instruction's 16, and lanes
    // 16-31 of each half the upper 16 of its 32 columns.
    const int a16 = lane & 15;
    const uint32_t at_l = ((lane >> 5) * 8 + (a16 >> 2)) * (TN * 2) + ((lane >> 4) & 1) * 32 + (a16 & 3) * 8;
    const auto turned = [&](int buf, int t, int piece) NKMX_INLINE {  // 4 tokens from t of a column of the piece
        const char* p = reinterpret_cast<const char*>(left[buf]) + at_l + ((piece ^ ((a16 >> 2) & TURN)) * 64) + t * (TN * 2);
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShorts)p);
    };
    const auto take_b = [&](bf16x8 (&b)[FK], int buf, int h) NKMX_INLINE {
#pragma unroll
        for (int j = 0; j < FK; ++j) {
            const uint32_t c = wk + 32 * j + r;
            b[j] = __builtin_bit_cast(bf16x8, right[buf][c * SLOTS + ((2 * h + g) ^ swizzle_t<SLOTS>(c))]);
        }
    };
    const auto take_a = [&](bf16x8& a, int buf, int h, int i) NKMX_INLINE {
        const s16x4 lo = turned(buf, 16 * h, wn / 32 + i), hi = turned(buf, 16 * h + 4, wn / 32 + i);
        const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
        const u32x4 both = {l2[0], l2[1], h2[0], h2[1]};
        a = __builtin_bit_cast(bf16x8, both);
    };
    // Sums of dy's columns, in the tiles of the first columns of x: a wave sums its tokens, a lane TN / 64 columns.
    float sum_dy[TN / 64] = {};
    const auto add_up = [&](int buf) NKMX_INLINE {
        const bf16x2 ones = {(bf16)1.0f, (bf16)1.0f};
#pragma unroll
        for (int j = 0; j < TN / 64; ++j)
#pragma unroll
            for (int t = 0; t < ROWS; t += 4) {
                const int piece = 2 * j + (lane >> 5);
                const char* p = reinterpret_cast<const char*>(left[buf]) + (wave * ROWS + t + (a16 >> 2)) * (TN * 2) +
                                ((piece ^ ((a16 >> 2) & TURN)) * 64) + ((lane >> 4) & 1) * 32 + (a16 & 3) * 8;
                const u32x2 four = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShorts)p));
                const uint32_t lo = four[0], hi = four[1];
                sum_dy[j] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, lo), ones, sum_dy[j], false);
                sum_dy[j] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, hi), ones, sum_dy[j], false);
            }
    };

    bf16x8 a[FN], b[2][FK];
    bf16x8 all_a[SHORT ? GROUPS : 1][FN], all_b[SHORT ? GROUPS : 1][FK];  // SHORT: a whole stage's operands
    const auto take_all = [&](int lb, int rb) NKMX_INLINE {
#pragma unroll
        for (int h = 0; h < GROUPS; ++h) {
            take_b(all_b[h], rb, h);
#pragma unroll
            for (int i = 0; i < FN; ++i) take_a(all_a[h][i], lb, h, i);
        }
    };
    // The 16 tokens h of a stage.  An operand is read for the next 16 as soon as it has been used (READS; after the last of
    // a stage: the next stage's first, in the other buffer); those reads and the instructions of what `work` adds go
    // between the matrix instructions.
    const auto tokens = [&](int from_left, int from_right, auto index, auto reads, auto work) NKMX_INLINE {
        constexpr int h = decltype(index)::value, then = (h + 1) % GROUPS;
        constexpr bool READS = decltype(reads)::value;
        if constexpr (READS) take_b(b[(h + 1) & 1], from_right, then);
#pragma unroll
        for (int i = 0; i < FN; ++i) {
#pragma unroll
            for (int j = 0; j < FK; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[h & 1][j], acc[i][j], 0, 0, 0);
            if constexpr (READS) take_a(a[i], from_left, then, i);
        }
        work();
#pragma unroll
        for (int z = 0; z < FN * FK; ++z) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
            __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);  // others
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // an LDS write
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto begin = [&](int buf) NKMX_INLINE {
        if constexpr (SHORT) return take_all(buf, buf);
        take_b(b[0], buf, 0);
#pragma unroll
        for (int i = 0; i < FN; ++i) take_a(a[i], buf, 0, i);
    };
    typedef std::integral_constant<int, 0> H0;
    typedef std::integral_constant<int, 1> H1;
    typedef std::integral_constant<int, 2> H2;
    typedef std::integral_constant<int, 3> H3;
    const auto run = [&](auto sums) NKMX_INLINE {
        Unit now, next;  // codes of the next stage and of the one after
        float scale[8];
        // A stage with dy in left[lb], codes turned in right[rb].  NEXT: another one follows; LOAD_X: and one after that, whose
        // codes are asked for; LOAD_D: dy of the stage DEPTH - 1 further on is.
        const auto stage = [&](uint32_t s, int lb, int rb, auto load_d, auto load_x, auto has_next) NKMX_INLINE {
            constexpr bool LOAD_D = decltype(load_d)::value, LOAD_X = decltype(load_x)::value, NEXT = decltype(has_next)::value;
            typedef std::integral_constant<bool, true> Reads;
            const int next_lb = lb + 1 == DEPTH ? 0 : lb + 1;
            // SHORT: the next stage's codes are waited for before anything new is asked for: the compiler counts the loads that may
            // still be on their way, and those to LDS, which it does not know, would have to arrive as well
            if constexpr (SHORT && NEXT) {
                if (has_x) settle(now);
            }
            if constexpr (LOAD_D) fetch_d(s + DEPTH - 1, lb ? lb - 1 : DEPTH - 1);
            if constexpr (ALL_X) {
                if constexpr (LOAD_X) fetch_x(next, s + 2);
                if constexpr (NEXT) spread_scales(now.e, scale);
            } else if (NEXT && has_x) {
                if constexpr (LOAD_X) fetch_x(next, s + 2);
                spread_scales(now.e, scale);
#pragma unroll
                for (int j = 0; j < 4; ++j) put_x(now, scale, rb ^ 1, j);
            }
            if constexpr (decltype(sums)::value) add_up(lb);
            if constexpr (SHORT) {
#pragma unroll
                for (int h = 0; h < GROUPS; ++h)
#pragma unroll
                    for (int i = 0; i < FN; ++i)
#pragma unroll
                        for (int j = 0; j < FK; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(all_a[h][i], all_b[h][j], acc[i][j], 0, 0, 0);
                if constexpr (LOAD_D && LOAD_X) {
                    if (has_x) arrived<(DEPTH - 2) * LOADS + (DEPTH - 1) * 8>();
                    else arrived<(DEPTH - 2) * LOADS>();
                } else {
                    arrived();
                }
                if constexpr (NEXT) take_all(next_lb, rb ^ 1);
                if constexpr (LOAD_X) now = next;
                return;
            }
            __builtin_amdgcn_sched_barrier(0);
            const auto turn = [&](int from, int to) NKMX_INLINE {
                if constexpr (ALL_X && NEXT) {
#pragma unroll
                    for (int j = from; j < to; ++j) put_x(now, scale, rb ^ 1, j);
                }
            };
            tokens(lb, rb, H0{}, Reads{}, [&]() NKMX_INLINE { turn(0, 1); });
            tokens(lb, rb, H1{}, Reads{}, [&]() NKMX_INLINE { turn(1, 2); });
            tokens(lb, rb, H2{}, Reads{}, [&]() NKMX_INLINE { turn(2, 4); });
            // This stage has been read and the next one is there: its codes turned, its dy arrived when no more than the loads
            // that were asked for behind it are on their way: dy of DEPTH - 2 stages, and 9 loads of codes (8, to be safe) each
            // and with its own.
            if constexpr (LOAD_D && LOAD_X) {
                if (has_x) arrived<(DEPTH - 2) * LOADS + (DEPTH - 1) * 8>();
                else arrived<(DEPTH - 2) * LOADS>();
            } else {
                arrived();
            }
            tokens(next_lb, rb ^ 1, H3{}, std::integral_constant<bool, NEXT>{}, [] {});
            if constexpr (LOAD_X) now = next;
        };
        typedef std::true_type Yes;
        typedef std::false_type No;
        const uint32_t fast = max(first, min(last, safe / BT));  // stages of whole tiles
        if (first < fast) {
            for (uint32_t s = 0; s + 1 < DEPTH && first + s < fast; ++s) fetch_d(first + s, s);
            if (has_x) {
                fetch_x(now, first);
                spread_scales(now.e, scale);
#pragma unroll
                for (int j = 0; j < 4; ++j) put_x(now, scale, 0, j);
                if (first + 1 < fast) fetch_x(now, first + 1);
            }
            arrived();
            begin(0);
            int lb = 0, rb = 0;
            const auto on = [&]() NKMX_INLINE {
                lb = lb + 1 == DEPTH ? 0 : lb + 1;
                rb ^= 1;
            };
            uint32_t s = first;
            for (; s + max(DEPTH - 1, 2) < fast; ++s, on()) stage(s, lb, rb, Yes{}, Yes{}, Yes{});
            if constexpr (DEPTH > 2)
                for (; s + 2 < fast; ++s, on()) stage(s, lb, rb, No{}, Yes{}, Yes{});
            if (s + 1 < fast) {
                stage(s, lb, rb, std::integral_constant<bool, DEPTH == 2>{}, No{}, Yes{});
                on();
            }
            stage(fast - 1, lb, rb, No{}, No{}, No{});
        }
#pragma unroll 1
        for (uint32_t s = fast; s < last; ++s) {  // the last tokens
            copy_d(s, 0);
            if (has_x) {
                copy_x(now, s);
                spread_scales(now.e, scale);
#pragma unroll
                for (int j = 0; j < 4; ++j) put_x(now, scale, 0, j);
            }
            arrived();
            begin(0);
            stage(s, 0, 0, No{}, No{}, No{});
        }
    };
    if (db != nullptr && tc == 0) run(std::true_type{});
    else run(std::false_type{});

    store_gradient<FN, FK>(acc, dw + blockIdx.y * part_stride, lddw, tr * TN + wn, tc * TK + wk, n, k, accumulate, r, g);
    if (db != nullptr && tc == 0) {  // the waves' sums of a column, joined in order
        float* part = reinterpret_cast<float*>(&right[0][0]);
#pragma unroll
        for (int j = 0; j < TN / 64; ++j) part[wave * TN + 64 * j + lane] = sum_dy[j];
        __syncthreads();
        for (int c = tid; c < TN; c += NT)
            if (tr * TN + c < n) {
                float s = part[c];
#pragma unroll
                for (int i = 1; i < WAVES; ++i) s += part[i * TN + c];
                float* p = db + blockIdx.y * part_stride_db + tr * TN + c;
                *p = accumulate ? *p + s : s;
            }
    }
}

// db alone (k = 0): sums of dy's columns.  A row of a tile is `lanes` lanes of 16 bytes, a power of two up to 64 that fits n, so
// that narrow matrices still fill the wave with rows; a thread adds up every 256 / lanes-th row of its part of t, eight loads
// on their way at a time, and the threads of a column are joined in order.  Bound by memory and by waits where few columns leave
// few workgroups: with the join of the parts 16384 x 4096 bf16 (134 MB) 43 us, 16384 x 1023 50, 200000 x 64 26.
template <typename T>
__global__ __launch_bounds__(256) void column_sums_kernel(float* db, const T* dy, uint64_t lddy, uint32_t t_rows, uint32_t n,
                                                          uint32_t lanes, uint32_t col_tiles, uint32_t rows_each,
                                                          uint32_t accumulate, uint64_t part_stride)
{
    constexpr int E = Lanes<T>::E;
    __shared__ float sums[256 * E];
    const uint32_t groups = 256 / lanes, lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
    const uint32_t tile = blockIdx.x % col_tiles, part = blockIdx.x / col_tiles;
    const uint32_t first = part * rows_each, last = min(t_rows, first + rows_each);
    const uint64_t col = ((uint64_t)tile * lanes + lane) * E;
    const int64_t live = (int64_t)n - (int64_t)col;
    float s[E] = {};
    for (uint64_t t = first + group; t < last; t += 8 * groups) {
        typename Pack<T, E>::vec v[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            v[i] = load_pack<T, E>(dy + (t + i * groups) * lddy + col, t + i * groups < last ? live : 0);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < E; ++j) s[j] += number(v[i][j]);
    }
#pragma unroll
    for (int j = 0; j < E; ++j) sums[threadIdx.x * E + j] = s[j];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < lanes * E; i += 256) {
        float sum = sums[i];
        for (uint32_t g = 1; g < groups; ++g) sum += sums[g * lanes * E + i];
        const uint64_t c = (uint64_t)tile * lanes * E + i;
        if (c < n) {
            float* p = db + part * part_stride + c;
            *p = accumulate ? *p + sum : sum;
        }
    }
}

// Joins the parts of a split weight gradient in order: dw, [parts][rows][ldp] in the workspace, and behind each part's
// dw its db as a row of `rows` numbers.  Rows of the workspace are whole quads.  4 parts of 4096 x 1024 (84 MB) 12 .. 13
// us = 6.5 TB/s.
__global__ __launch_bounds__(256) void join_parts_kernel(float* dw, uint64_t lddw, float* db, const float* part, uint32_t parts,
                                                         uint64_t part_stride, uint32_t rows, uint32_t cols, uint64_t ldp,
                                                         uint32_t accumulate)
{
    const uint32_t per_row = (cols + 3) / 4;
    uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint64_t quads = (uint64_t)rows * per_row;
    float* o;
    int64_t live;
    if (i < quads) {
        const uint64_t row = i / per_row;
        const uint32_t col = (uint32_t)(i - row * per_row) * 4;
        part += row * ldp + col;
        o = dw + row * lddw + col;
        live = (int64_t)cols - (int64_t)col;
    } else {
        i -= quads;
        live = (int64_t)rows - (int64_t)(4 * i);
        if (db == nullptr || live <= 0) return;
        part += rows * ldp + 4 * i;
        o = db + 4 * i;
    }
    f32x4 s = *reinterpret_cast<const f32x4*>(part);
    uint32_t p = 1;
    for (; p + 4 <= parts; p += 4) {  // four loads on their way at a time, added in order
        f32x4 v[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const f32x4*>(part + (p + j) * part_stride);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) s += v[j];
    }
    for (; p < parts; ++p) s += *reinterpret_cast<const f32x4*>(part + p * part_stride);
    if (accumulate) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < live) s[j] = o[j] + s[j];
    }
    store_pack<float, 4>(o, s, live);
}

// ---------------------------------------------------------------- host side

// hipLaunchKernel returns what THIS launch did; the runtime's "last error" is left alone unless the launch
// failed (then it is cleared, since the failure is reported through the return value).
template <typename Tuple, size_t... I>
inline void arg_pointers(Tuple& vals, void** out, std::index_sequence<I...>)
{
    ((out[I] = static_cast<void*>(&std::get<I>(vals))), ...);
}

constexpr uint64_t kMaxThreads = 1ull << 32;  // the runtime takes grids of fewer threads in a dimension

template <typename... KArgs, typename... Args>
inline int launch(void (*kernel)(KArgs...), dim3 grid, uint32_t block, hipStream_t s, Args... args)
{
    static_assert(sizeof...(KArgs) == sizeof...(Args), "kernel argument count");
    std::tuple<KArgs...> vals(static_cast<KArgs>(args)...);
    void* ptrs[sizeof...(KArgs)];
    arg_pointers(vals, ptrs, std::index_sequence_for<KArgs...>{});
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(block), ptrs, 0, s);
    if (e != hipSuccess) (void)hipGetLastError();
    return e == hipSuccess ? NKMX_OK : (int)e;
}

constexpr uint64_t kMaxSize = 0x7FFFFFFFull;
inline uint64_t steps_of(uint64_t cols) { return (cols + kStep - 1) / kStep; }
inline uint64_t size_of(int type) { return type == NKMX_F32 ? 4 : 2; }
inline bool known_type(int type) { return type == NKMX_F32 || type == NKMX_BF16 || type == NKMX_F16; }
inline bool on(const void* p, uint64_t align) { return (reinterpret_cast<uintptr_t>(p) & (align - 1)) == 0; }

// A buffer of a call: rows of `width` bytes, `pitch` apart.
struct Area {
    uintptr_t at;
    uint64_t rows, width, pitch;
};
inline Area area(const void* p, uint64_t rows, uint64_t cols, uint64_t ld, uint64_t size)
{
    return Area{reinterpret_cast<uintptr_t>(p), rows, cols * size, ld * size};
}
inline Area run(const void* p, uint64_t bytes) { return Area{reinterpret_cast<uintptr_t>(p), 1, bytes, bytes}; }

// Whether two buffers share a byte.  Two matrices with the same leading dimension may interleave (column
// ranges of one larger matrix); otherwise the whole extents count.
inline bool overlap(const Area& a, const Area& b)
{
    if (!a.rows || !b.rows || !a.width || !b.width) return false;
    const uintptr_t ea = a.at + (a.rows - 1) * a.pitch + a.width, eb = b.at + (b.rows - 1) * b.pitch + b.width;
    if (ea <= b.at || eb <= a.at) return false;
    if (a.rows > 1 && b.rows > 1 && a.pitch == b.pitch) {
        const uint64_t off = b.at >= a.at ? (b.at - a.at) % a.pitch : (a.pitch - (a.at - b.at) % a.pitch) % a.pitch;
        return !(off >= a.width && off + b.width <= a.pitch);
    }
    return true;
}
inline bool same(const Area& a, const Area& b)
{
    return a.at == b.at && a.rows == b.rows && a.width == b.width && (a.rows <= 1 || a.pitch == b.pitch);
}

// Calls f with a null pointer of the element type.
template <typename F>
inline int for_type(int type, F f)
{
    switch (type) {
        case NKMX_F32: return f((float*)nullptr);
        case NKMX_BF16: return f((bf16*)nullptr);
        default: return f((f16*)nullptr);
    }
}

// The streaming launches: steps of the packed matrix, lanes, workgroups.
struct Stream {
    FastDiv steps;
    uint32_t n_steps, cols, blocks;
};
template <typename T, int U>
inline bool stream_of(Stream& s, uint64_t rows, uint64_t cols)
{
    const uint64_t steps = steps_of(cols), total = rows * steps;  // both below 2^31
    if (total > 0xFFFFFFFFull) return false;
    const uint64_t blocks = (total * Lanes<T>::step + 256 * U - 1) / (256 * U);
    if (blocks > kMaxSize) return false;
    s = Stream{fast_div((uint32_t)steps), (uint32_t)total, (uint32_t)cols, (uint32_t)blocks};
    return true;
}

// The grid of a streaming launch: one row of workgroups, or several where that would be too many threads (from 2^34 fp32 numbers on).
inline dim3 stream_grid(const Stream& s)
{
    if ((uint64_t)s.blocks * 256 < kMaxThreads) return dim3(s.blocks);
    return dim3(kGridRow, (s.blocks - 1) / kGridRow + 1);
}

// The rules on matrices of numbers: sizes, leading dimension, alignment.
inline int check_matrix(const void* p, int type, uint64_t rows, uint64_t cols, uint64_t ld)
{
    if (rows > kMaxSize || cols > kMaxSize || ld > kMaxSize || (rows > 1 && ld < cols)) return NKMX_ERANGE;
    if (rows == 0 || cols == 0) return NKMX_OK;
    if (!p) return NKMX_ENULL;
    return on(p, size_of(type)) ? NKMX_OK : NKMX_EALIGN;
}
inline int check_packed(const void* codes, const void* scales, uint64_t rows, uint64_t cols)
{
    if (rows > kMaxSize || cols > kMaxSize) return NKMX_ERANGE;
    if (rows == 0 || cols == 0) return NKMX_OK;
    if (!codes || !scales) return NKMX_ENULL;
    return on(codes, 16) && on(scales, 4) ? NKMX_OK : NKMX_EALIGN;
}
inline Area codes4(const void* p, uint64_t rows, uint64_t cols) { return run(p, rows * steps_of(cols) * kStepBytes4); }
inline Area codes8(const void* p, uint64_t rows, uint64_t cols) { return run(p, rows * steps_of(cols) * kStep); }
inline Area scale_bytes(const void* p, uint64_t rows, uint64_t cols) { return run(p, rows * steps_of(cols) * 4); }

#define NKMX_TRY(call)                 \
    do {                               \
        const int rc_ = (call);        \
        if (rc_ != NKMX_OK) return rc_; \
    } while (0)

// ---- product

// A tile's rows lie within the 4 GB that a buffer load can address: 256 rows of k / 2 bytes.
constexpr uint64_t kTilesMaxK = 1ull << 24;
// Whether x is quantized inside the product: every workgroup (16 rows of b) then quantizes all of x, 100 instructions a
// step of k and wave, which a launch saved pays for while b is small (us, inside / before, captured): 1 x 4096 x 1024 3.0 /
// 4.3, 8 x 1024 x 4096 5.9 / 5.8, 1 x 8192 x 8192 12.6 / 10.4.  A call made eagerly saves 4 us of host time as well.
inline bool quantizes_inside(uint64_t m, uint64_t n, uint64_t k) { return m <= 8 && k && n * k <= 1ull << 24; }

template <typename T, int MT, int NT, bool FUSED>
inline int launch_rows(T* y, uint64_t ldy, const T* x, uint64_t ldx, const uint8_t* ca, const uint8_t* sa,
                       const uint8_t* cb, const uint8_t* sb, const T* bias, uint64_t m, uint64_t n, uint64_t k,
                       hipStream_t s)
{
    const uint64_t blocks = ((n + 16 * NT - 1) / (16 * NT)) * ((m + 16 * MT - 1) / (16 * MT));
    if (blocks * (64 * kRowsWaves) >= kMaxThreads) return NKMX_ERANGE;
    if (!y) return NKMX_OK;
    return launch(mx4_rows_kernel<T, MT, NT, FUSED>, dim3((uint32_t)blocks), 64 * kRowsWaves, s, y, ldy, x, ldx, ca, sa, cb, sb, bias,
                  (uint32_t)m, (uint32_t)n, (uint32_t)k, (uint32_t)steps_of(k));
}

template <typename T, int TM, int TN, int WM, int WN, int BUFFERS>
inline int launch_tiles(T* y, uint64_t ldy, const uint8_t* ca, const uint8_t* sa, const uint8_t* cb, const uint8_t* sb,
                        const T* bias, uint64_t m, uint64_t n, uint64_t k, hipStream_t s)
{
    const uint64_t rt = (m + TM - 1) / TM, ct = (n + TN - 1) / TN;
    if (rt * ct * (64 * (TM / WM) * (TN / WN)) >= kMaxThreads) return NKMX_ERANGE;
    if (!y) return NKMX_OK;
    return launch(mx4_tiles_kernel<T, TM, TN, WM, WN, BUFFERS>, dim3((uint32_t)(rt * ct)), 64 * (TM / WM) * (TN / WN), s, y, ldy,
                  ca, sa, cb, sb, bias, (uint32_t)m, (uint32_t)n, (uint32_t)steps_of(k), (uint32_t)rt, (uint32_t)ct);
}

// Which kernel, by counts of workgroups (us at m x n x k, codes from HBM):
//   rows 16 x 16      up to 16 rows, and while there are at most 384 of them: 64 x 1024 x 4096 4.8 against 8.0 by tiles,
//                     100 x 1024 x 1024 (448) 4.2 against 4.4, 200 x 1024 x 1024 (832) 6.6 against 4.4
//   rows 32 x 32      up to 32 rows: 32 x 8192 x 8192 13.1 against 15.3 by tiles of 64, and 22.7 by rows of 16
//   tiles 256         from 192 tiles: 4096^3 43 against 55 by tiles of 128; 2048 x 4096 x 4096 (128 tiles) 33 against 26
//   tiles 128         from 192 tiles: 1024 x 4096 x 4096 17 against 22 by tiles of 64; 512 x 4096 x 4096 (128) 15 against
//                     12.6; with four buffers while every workgroup has a CU of its own (512 x 8192 x 8192 30 against 41
//                     with two), with two beyond (2048 x 4096 x 4096 26.6 against 30.3)
//   tiles 64 x 32     up to 128 tiles of 64: 64 x 8192 x 8192 15.0 against 17.2, but 128 x 8192 x 8192 21 against 17
// Without y nothing is launched: whether the launch is one that the runtime takes.
template <typename T>
int product(T* y, uint64_t ldy, const uint8_t* ca, const uint8_t* sa, const uint8_t* cb, const uint8_t* sb,
            const T* bias, uint64_t m, uint64_t n, uint64_t k, hipStream_t s)
{
    const auto tiles = [&](uint64_t side) { return ((m + side - 1) / side) * ((n + side - 1) / side); };
    const T* none = nullptr;
    if (m <= 16 || tiles(16) <= 384) return launch_rows<T, 1, 1, false>(y, ldy, none, 0, ca, sa, cb, sb, bias, m, n, k, s);
    if (k == 0 || m <= 32 || k > kTilesMaxK)
        return launch_rows<T, 2, 2, false>(y, ldy, none, 0, ca, sa, cb, sb, bias, m, n, k, s);
    if (tiles(256) >= 192) return launch_tiles<T, 256, 256, 128, 64, 2>(y, ldy, ca, sa, cb, sb, bias, m, n, k, s);
    if (tiles(128) > 256) return launch_tiles<T, 128, 128, 64, 64, 2>(y, ldy, ca, sa, cb, sb, bias, m, n, k, s);
    if (tiles(128) >= 192) return launch_tiles<T, 128, 128, 64, 64, 4>(y, ldy, ca, sa, cb, sb, bias, m, n, k, s);
    if (tiles(64) > 128) return launch_tiles<T, 64, 64, 32, 32, 4>(y, ldy, ca, sa, cb, sb, bias, m, n, k, s);
    return launch_tiles<T, 64, 32, 32, 32, 4>(y, ldy, ca, sa, cb, sb, bias, m, n, k, s);
}

// ---- weight gradient

struct WgradPlan {
    int side;              // tile: 256, 128 or 64; 0: no columns, db alone, by tiles of `lanes` times 16 bytes of a row
    uint32_t lanes;
    uint64_t row_tiles, col_tiles, parts, stages_each, ldp;
    uint64_t part_floats;  // of dw and db of one part in the workspace
};

WgradPlan wgrad_plan(int type, uint64_t t, uint64_t n, uint64_t k)  // n > 0
{
    const auto tiles = [&](uint64_t side) { return ((n + side - 1) / side) * ((k + side - 1) / side); };
    WgradPlan p = {};
    if (k == 0) {
        // db alone: t is cut until there are two workgroups for every CU while a thread has 16 rows, in at most 64 parts, whose
        // join waits 0.12 us for each
        const uint64_t per_lane = 16 / size_of(type), wanted = (n + per_lane - 1) / per_lane;
        p.lanes = 1;
        while (p.lanes < 64 && p.lanes < wanted) p.lanes *= 2;
        p.row_tiles = (wanted + p.lanes - 1) / p.lanes;
        const uint64_t most = t / (256 / p.lanes * 16), fill = 512 / p.row_tiles;
        p.parts = most < fill ? most : fill;
        p.parts = p.parts < 1 ? 1 : p.parts > 64 ? 64 : p.parts;
        p.stages_each = (t + p.parts - 1) / p.parts;
        p.part_floats = (n + 3) / 4 * 4;
        return p;
    }
    // Tiles of 256 where they, cut along 1024 tokens, give every CU one (bf16, us with tiles of 256 / 128 / 64: 16384 x 1024
    // x 1024 56 / 70 / 88, 2048 x 4096 x 4096 74 / 94 / 152).  Else of 128 where nearly every CU has one without a cut (500 x
    // 2000 x 2000 bf16 20 against 25 with tiles of 64, fp32 27 against 33; 1000 x 1000 x 1000 bf16 23 against 16.3), and for
    // the other types, whose tiles of 64 have no deep buffers, also where they give every CU one cut along 512 (fp32 3000 x
    // 1000 x 1000 39.7 against 43.7, 1000 x 1000 x 1000 29 against 22.7)
    const bool small = tiles(128) < 192 && (type == NKMX_BF16 || tiles(128) * ((t + 511) / 512) <= 256);
    p.side = tiles(256) * ((t + 1023) / 1024) >= 256 ? 256 : (small ? 64 : 128);
    const uint64_t bt = p.side == 256 && type != NKMX_BF16 ? 32 : 64;
    const uint64_t stages = (t + bt - 1) / bt;
    p.row_tiles = (n + p.side - 1) / p.side;
    p.col_tiles = (k + p.side - 1) / p.side;
    const uint64_t count = p.row_tiles * p.col_tiles;
    // split t until the tiles fill the chip, but keep 8 stages a part
    uint64_t parts = 256 / count;
    // More tiles than CUs: their last round may leave most CUs idle.  Cut in parts the rounds come out evenly, which is
    // weighed against writing and joining the parts: a tile of 256 takes 25, 50, 70 ns a token (bf16, fp16, fp32), a part
    // 1.8 ps a number (16384 x 4352 x 4096, 272 tiles: bf16 816 us whole, 645 in 3 parts, fp32 2322 and 1551 in 4; 16384 x
    // 5120 x 5120, 400 tiles, bf16: 881 whole, 929 in 2, 883 in 3).
    if (p.side == 256 && count > 256) {
        const double token = type == NKMX_BF16 ? 25e-3 : type == NKMX_F16 ? 50e-3 : 70e-3;
        double best = 0;
        for (uint64_t q = 1; q <= 4; ++q) {
            const double us = (double)((count * q + 255) / 256) / (double)q * (double)t * token +
                              (q > 1 ? (double)q * (double)n * (double)k * 1.8e-6 : 0.0);
            if (q == 1 || us < best) {
                best = us;
                parts = q;
            }
        }
    }
    if (p.side == 64) {
        // A stage of a tile of 64 is mostly waiting, which two or three workgroups on a CU share (it takes 0.62, 0.9, 1.2 us, and
        // 40 % more for each further one); against that stand 3 us for the join, 0.12 for each part's wait in it and the
        // parts' bytes: 16384 x 300 x 500 bf16 (40 tiles) 12 parts 29.6, 24 30.8, 8 38; 1000 x 1000 x 1000 (256 tiles) whole
        // 17.4, 3 parts 20.8; 1024 x 512 x 512 (64 tiles) whole 13.9, 4 parts 11.4.
        const double stage = type == NKMX_BF16 ? 0.62 : type == NKMX_F16 ? 0.9 : 1.2;
        const uint64_t resident = type == NKMX_F32 ? 2 : 3;
        double best = 0;
        parts = 1;
        for (uint64_t q = 1; q == 1 || (q * count <= 256 * resident && q * 4 <= stages && q <= 64); ++q) {
            const double us = (double)((stages + q - 1) / q) * stage * (1.0 + 0.4 * (double)((q * count - 1) / 256)) +
                              (q > 1 ? 3.0 + (double)q * (0.12 + (double)n * (double)k * 1.2e-6) : 0.0);
            if (q == 1 || us < best) {
                best = us;
                parts = q;
            }
        }
    } else if (parts > stages / 8) {
        parts = stages / 8;
    }
    if (parts < 1) parts = 1;
    p.stages_each = (stages + parts - 1) / parts;
    p.parts = p.stages_each ? (stages + p.stages_each - 1) / p.stages_each : 1;
    if (p.parts < 1) p.parts = 1;
    p.ldp = (k + 3) / 4 * 4;
    p.part_floats = n * p.ldp + (n + 3) / 4 * 4;
    return p;
}

inline uint64_t workspace_of(const WgradPlan& p) { return p.parts > 1 ? p.parts * p.part_floats * 4 : 0; }

template <typename T, int TN, int TK, int WN, int WK, int BT>
inline int launch_wgrad(const WgradPlan& p, float* dw, uint64_t lddw, float* db, const T* dy, uint64_t lddy,
                        const uint8_t* codes, const uint8_t* scales, uint64_t t, uint64_t n, uint64_t k,
                        uint32_t accumulate, uint64_t stride, hipStream_t s)
{
    const uint64_t tiles = p.row_tiles * p.col_tiles;
    if (tiles * (64 * (TN / WN) * (TK / WK)) >= kMaxThreads) return NKMX_ERANGE;
    const auto with = [&](auto kernel) {
        return launch(kernel, dim3((uint32_t)tiles, (uint32_t)p.parts), 64 * (TN / WN) * (TK / WK), s, dw, lddw, db, dy, lddy,
                      codes, scales, (uint32_t)t, (uint32_t)n, (uint32_t)k, (uint32_t)steps_of(k), (uint32_t)p.row_tiles,
                      (uint32_t)p.col_tiles, (uint32_t)p.stages_each, accumulate, stride, stride);
    };
    if constexpr (std::is_same_v<T, bf16>) {
        if (on(dy, 4) && lddy % 2 == 0 && lddy < (1u << 24)) return with(act8_wgrad_raw_kernel<TN, TK, WN, WK>);
    }
    return with(act8_wgrad_kernel<T, TN, TK, WN, WK, BT>);
}

}  // namespace

extern "C" {

int nkmx_version(void) { return NKMX_VERSION; }

const char* nkmx_strerror(int code)
{
    switch (code) {
        case NKMX_OK: return "success";
        case NKMX_ENULL: return "nkmx: a required pointer is NULL";
        case NKMX_EALIGN: return "nkmx: a pointer is not aligned (codes 16 bytes, scales 4, numbers their size)";
        case NKMX_ERANGE: return "nkmx: a size, leading dimension, type or activation is out of range";
        case NKMX_EALIAS: return "nkmx: an output overlaps another buffer of the call";
        case NKMX_EWORK: return "nkmx: the workspace is missing, too small or not on a 16-byte boundary";
        default: break;
    }
    if (code > 0) return hipGetErrorString((hipError_t)code);
    return "nkmx: unknown error";
}

int nkmx_mx4_quantize(const void* x, int type, uint64_t rows, uint64_t cols, uint64_t ldx, uint8_t* codes,
                      uint8_t* scales, int transpose, void* stream)
{
    if (!known_type(type)) return NKMX_ERANGE;
    NKMX_TRY(check_matrix(x, type, rows, cols, ldx));
    if (rows == 0 || cols == 0) return NKMX_OK;
    const uint64_t pr = transpose ? cols : rows, pc = transpose ? rows : cols;  // of the packed matrix
    NKMX_TRY(check_packed(codes, scales, pr, pc));
    const Area ax = area(x, rows, cols, ldx, size_of(type)), ac = codes4(codes, pr, pc), as = scale_bytes(scales, pr, pc);
    if (overlap(ax, ac) || overlap(ax, as) || overlap(ac, as)) return NKMX_EALIAS;
    const hipStream_t s = (hipStream_t)stream;
    return for_type(type, [&](auto* null) -> int {
        typedef std::remove_pointer_t<decltype(null)> T;
        if (transpose) {
            // 8 bytes a lane and row from 1024 workgroups on (8192 x 4096 fp32 25.8 us against 28.6 with 4), 4 below
            // (1024 x 1024 5.9 against 7.4)
            const auto with = [&](auto bytes) -> int {
                constexpr int CPL = decltype(bytes)::value / (int)sizeof(T);
                const uint64_t tiles = (cols + 64 * CPL - 1) / (64 * CPL), bands = (rows + 255) / 256;
                if (tiles * bands * 512 >= kMaxThreads) return NKMX_ERANGE;
                return launch(mx4_quantize_transposed_kernel<T, CPL>, dim3((uint32_t)(tiles * bands)), 512, s, (const T*)x, ldx,
                              codes, scales, (uint32_t)rows, (uint32_t)cols, (uint32_t)steps_of(rows), (uint32_t)tiles);
            };
            if ((rows + 255) / 256 * ((cols * sizeof(T) + 511) / 512) >= 1024) return with(std::integral_constant<int, 8>{});
            return with(std::integral_constant<int, 4>{});
        }
        Stream g;
        // four pieces a lane where that still fills the chip: a pass that mostly reads wants more in flight than its
        // lanes' 16 bytes (16384 x 8192 bf16 58 us with one, 55 with two, 52.5 with four; passes that write as much
        // as they read lose by it)
        if (!stream_of<T, 4>(g, rows, cols)) return NKMX_ERANGE;
        if (g.blocks >= 1024)
            return launch(mx4_quantize_kernel<T, 4>, stream_grid(g), 256, s, (const T*)x, ldx, codes, scales, g.steps,
                          g.n_steps, g.cols);
        stream_of<T, 1>(g, rows, cols);
        return launch(mx4_quantize_kernel<T, 1>, stream_grid(g), 256, s, (const T*)x, ldx, codes, scales, g.steps, g.n_steps,
                      g.cols);
    });
}

int nkmx_mx4_dequantize(void* out, int type, uint64_t rows, uint64_t cols, uint64_t ldo, const uint8_t* codes,
                        const uint8_t* scales, void* stream)
{
    if (!known_type(type)) return NKMX_ERANGE;
    NKMX_TRY(check_matrix(out, type, rows, cols, ldo));
    NKMX_TRY(check_packed(codes, scales, rows, cols));
    if (rows == 0 || cols == 0) return NKMX_OK;
    const Area ao = area(out, rows, cols, ldo, size_of(type));
    if (overlap(ao, codes4(codes, rows, cols)) || overlap(ao, scale_bytes(scales, rows, cols))) return NKMX_EALIAS;
    return for_type(type, [&](auto* null) -> int {
        typedef std::remove_pointer_t<decltype(null)> T;
        Stream g;
        if (!stream_of<T, 1>(g, rows, cols)) return NKMX_ERANGE;
        return launch(mx4_dequantize_kernel<T, 1>, stream_grid(g), 256, (hipStream_t)stream, (T*)out, ldo, codes, scales,
                      g.steps, g.n_steps, g.cols);
    });
}

int nkmx_mx4_matmul(void* y, int type, uint64_t m, uint64_t n, uint64_t k, uint64_t ldy, const uint8_t* a_codes,
                    const uint8_t* a_scales, const uint8_t* b_codes, const uint8_t* b_scales, const void* bias,
                    void* stream)
{
    if (!known_type(type)) return NKMX_ERANGE;
    NKMX_TRY(check_matrix(y, type, m, n, ldy));
    if (m == 0 || n == 0) return NKMX_OK;
    NKMX_TRY(check_packed(a_codes, a_scales, m, k));
    NKMX_TRY(check_packed(b_codes, b_scales, n, k));
    if (bias && !on(bias, size_of(type))) return NKMX_EALIGN;
    const Area ay = area(y, m, n, ldy, size_of(type));
    if (overlap(ay, codes4(a_codes, m, k)) || overlap(ay, scale_bytes(a_scales, m, k)) ||
        overlap(ay, codes4(b_codes, n, k)) || overlap(ay, scale_bytes(b_scales, n, k)) ||
        (bias && overlap(ay, run(bias, n * size_of(type)))))
        return NKMX_EALIAS;
    return for_type(type, [&](auto* null) -> int {
        typedef std::remove_pointer_t<decltype(null)> T;
        return product<T>((T*)y, ldy, a_codes, a_scales, b_codes, b_scales, (const T*)bias, m, n, k, (hipStream_t)stream);
    });
}

uint64_t nkmx_mx4_linear_workspace(uint64_t m, uint64_t n, uint64_t k)
{
    if (m > kMaxSize || n == 0 || n > kMaxSize || k > kMaxSize || quantizes_inside(m, n, k)) return 0;
    return m * steps_of(k) * (kStepBytes4 + 4);
}

int nkmx_mx4_linear(void* y, const void* x, int type, uint64_t m, uint64_t n, uint64_t k, uint64_t ldy, uint64_t ldx,
                    const uint8_t* b_codes, const uint8_t* b_scales, const void* bias, void* workspace,
                    uint64_t workspace_bytes, void* stream)
{
    if (!known_type(type)) return NKMX_ERANGE;
    NKMX_TRY(check_matrix(y, type, m, n, ldy));
    NKMX_TRY(check_matrix(x, type, m, k, ldx));
    if (m == 0 || n == 0) return NKMX_OK;
    NKMX_TRY(check_packed(b_codes, b_scales, n, k));
    if (bias && !on(bias, size_of(type))) return NKMX_EALIGN;
    const uint64_t need = nkmx_mx4_linear_workspace(m, n, k);
    if (need && (!workspace || workspace_bytes < need || !on(workspace, 16))) return NKMX_EWORK;
    const Area ay = area(y, m, n, ldy, size_of(type)), ax = area(x, m, k, ldx, size_of(type)), aw = run(workspace, need);
    const Area ac = codes4(b_codes, n, k), as = scale_bytes(b_scales, n, k), ab = run(bias, bias ? n * size_of(type) : 0);
    if (overlap(ay, ax) || overlap(ay, ac) || overlap(ay, as) || overlap(ay, ab) || overlap(aw, ay) || overlap(aw, ax) ||
        overlap(aw, ac) || overlap(aw, as) || overlap(aw, ab))
        return NKMX_EALIAS;
    const hipStream_t s = (hipStream_t)stream;
    uint8_t* ca = (uint8_t*)workspace;
    uint8_t* sa = ca + m * steps_of(k) * kStepBytes4;
    if (need) {
        NKMX_TRY(product<float>(nullptr, 0, nullptr, nullptr, nullptr, nullptr, nullptr, m, n, k, s));
        NKMX_TRY(nkmx_mx4_quantize(x, type, m, k, ldx, ca, sa, 0, stream));
    }
    return for_type(type, [&](auto* null) -> int {
        typedef std::remove_pointer_t<decltype(null)> T;
        if (quantizes_inside(m, n, k))
            return launch_rows<T, 1, 1, true>((T*)y, ldy, (const T*)x, ldx, nullptr, nullptr, b_codes, b_scales,
                                           (const T*)bias, m, n, k, s);
        return product<T>((T*)y, ldy, ca, sa, b_codes, b_scales, (const T*)bias, m, n, k, s);
    });
}

int nkmx_act8_save(const void* x, void* y, int type, int fn, uint64_t rows, uint64_t cols, uint64_t ldx, uint64_t ldy,
                   uint8_t* codes, uint8_t* scales, void* stream)
{
    if (!known_type(type) || fn < NKMX_NONE || fn > NKMX_SILU) return NKMX_ERANGE;
    NKMX_TRY(check_matrix(x, type, rows, cols, ldx));
    if (fn != NKMX_NONE) NKMX_TRY(check_matrix(y, type, rows, cols, ldy));
    const bool saves = fn == NKMX_NONE || codes || scales;
    if (saves) NKMX_TRY(check_packed(codes, scales, rows, cols));
    if (rows == 0 || cols == 0) return NKMX_OK;
    const uint64_t b = size_of(type);
    const Area ax = area(x, rows, cols, ldx, b), ay = area(y, fn == NKMX_NONE ? 0 : rows, cols, ldy, b);
    const Area ac = codes8(codes, saves ? rows : 0, cols), as = scale_bytes(scales, saves ? rows : 0, cols);
    if (overlap(ac, ax) || overlap(as, ax) || overlap(ac, as) || overlap(ac, ay) || overlap(as, ay) ||
        (overlap(ay, ax) && !same(ay, ax)))
        return NKMX_EALIAS;
    return for_type(type, [&](auto* null) -> int {
        typedef std::remove_pointer_t<decltype(null)> T;
        Stream g;
        if (!stream_of<T, 1>(g, rows, cols)) return NKMX_ERANGE;
        const auto with = [&](auto kernel) {
            return launch(kernel, stream_grid(g), 256, (hipStream_t)stream, (const T*)x, ldx, (T*)y, ldy, codes, scales,
                          g.steps, g.n_steps, g.cols);
        };
        if (fn == NKMX_GELU) return with(act8_save_kernel<T, NKMX_GELU, 1>);
        if (fn == NKMX_SILU) return with(act8_save_kernel<T, NKMX_SILU, 1>);
        return with(act8_save_kernel<T, NKMX_NONE, 1>);
    });
}

static int act8_read(void* out, const void* dy, int type, int fn, uint64_t rows, uint64_t cols, uint64_t ldo,
                     uint64_t lddy, const uint8_t* codes, const uint8_t* scales, void* stream)
{
    NKMX_TRY(check_matrix(out, type, rows, cols, ldo));
    if (fn != NKMX_NONE) NKMX_TRY(check_matrix(dy, type, rows, cols, lddy));
    NKMX_TRY(check_packed(codes, scales, rows, cols));
    if (rows == 0 || cols == 0) return NKMX_OK;
    const uint64_t b = size_of(type);
    const Area ao = area(out, rows, cols, ldo, b), ad = area(dy, fn == NKMX_NONE ? 0 : rows, cols, lddy, b);
    if (overlap(ao, codes8(codes, rows, cols)) || overlap(ao, scale_bytes(scales, rows, cols)) ||
        (overlap(ao, ad) && !same(ao, ad)))
        return NKMX_EALIAS;
    return for_type(type, [&](auto* null) -> int {
        typedef std::remove_pointer_t<decltype(null)> T;
        Stream g;
        if (!stream_of<T, 1>(g, rows, cols)) return NKMX_ERANGE;
        const auto with = [&](auto kernel) {
            return launch(kernel, stream_grid(g), 256, (hipStream_t)stream, (T*)out, ldo, (const T*)dy, lddy, codes,
                          scales, g.steps, g.n_steps, g.cols);
        };
        if (fn == NKMX_GELU) return with(act8_grad_kernel<T, NKMX_GELU, 1>);
        if (fn == NKMX_SILU) return with(act8_grad_kernel<T, NKMX_SILU, 1>);
        return with(act8_grad_kernel<T, NKMX_NONE, 1>);
    });
}

int nkmx_act8_load(void* out, int type, uint64_t rows, uint64_t cols, uint64_t ldo, const uint8_t* codes,
                   const uint8_t* scales, void* stream)
{
    if (!known_type(type)) return NKMX_ERANGE;
    return act8_read(out, nullptr, type, NKMX_NONE, rows, cols, ldo, 0, codes, scales, stream);
}

int nkmx_act8_grad(void* dx, const void* dy, int type, int fn, uint64_t rows, uint64_t cols, uint64_t lddx,
                   uint64_t lddy, const uint8_t* codes, const uint8_t* scales, void* stream)
{
    if (!known_type(type) || (fn != NKMX_GELU && fn != NKMX_SILU)) return NKMX_ERANGE;
    return act8_read(dx, dy, type, fn, rows, cols, lddx, lddy, codes, scales, stream);
}

uint64_t nkmx_act8_wgrad_workspace(int type, uint64_t t, uint64_t n, uint64_t k)
{
    if (!known_type(type) || t > kMaxSize || n > kMaxSize || k > kMaxSize || n == 0) return 0;
    return workspace_of(wgrad_plan(type, t, n, k));
}

int nkmx_act8_wgrad(float* dw, float* db, const void* dy, int type, uint64_t t, uint64_t n, uint64_t k, uint64_t lddw,
                    uint64_t lddy, const uint8_t* codes, const uint8_t* scales, int accumulate, void* workspace,
                    uint64_t workspace_bytes, void* stream)
{
    if (!known_type(type)) return NKMX_ERANGE;
    NKMX_TRY(check_matrix(dw, NKMX_F32, n, k, lddw));
    NKMX_TRY(check_matrix(dy, type, t, n, lddy));
    NKMX_TRY(check_packed(codes, scales, t, k));
    if (db && !on(db, 4)) return NKMX_EALIGN;
    if (n == 0 || (k == 0 && !db)) return NKMX_OK;
    const WgradPlan p = wgrad_plan(type, t, n, k);
    const uint64_t need = workspace_of(p);
    if (need && (!workspace || workspace_bytes < need || !on(workspace, 16))) return NKMX_EWORK;
    const Area aw = area(dw, n, k, lddw, 4), ab = run(db, db ? n * 4 : 0), ad = area(dy, t, n, lddy, size_of(type));
    const Area ac = codes8(codes, t, k), as = scale_bytes(scales, t, k), ak = run(workspace, need);
    for (const Area* o : {&aw, &ab, &ak})
        if (overlap(*o, ad) || overlap(*o, ac) || overlap(*o, as)) return NKMX_EALIAS;
    if (overlap(aw, ab) || overlap(aw, ak) || overlap(ab, ak)) return NKMX_EALIAS;
    const hipStream_t s = (hipStream_t)stream;
    const bool split = p.parts > 1;
    const uint64_t join_blocks = (n * ((k + 3) / 4) + (db ? (n + 3) / 4 : 0) + 255) / 256;
    if (split && join_blocks * 256 >= kMaxThreads) return NKMX_ERANGE;
    float* part = (float*)workspace;
    float* to = split ? part : dw;
    float* to_db = !db ? nullptr : (split ? part + n * p.ldp : db);  // (ldp is 0 where there are no columns)
    const uint64_t ld = split ? p.ldp : lddw, stride = split ? p.part_floats : 0;
    const uint32_t add = !split && accumulate ? 1u : 0u;
    NKMX_TRY(for_type(type, [&](auto* null) -> int {
        typedef std::remove_pointer_t<decltype(null)> T;
        constexpr int BT = Parts<T>::count == 1 ? 64 : 32;
        if (p.side == 0)
            return launch(column_sums_kernel<T>, dim3((uint32_t)(p.row_tiles * p.parts)), 256, s, to_db, (const T*)dy, lddy,
                          (uint32_t)t, (uint32_t)n, p.lanes, (uint32_t)p.row_tiles, (uint32_t)p.stages_each, add, stride);
        if (p.side == 256)
            return launch_wgrad<T, 256, 256, 128, 64, BT>(p, to, ld, to_db, (const T*)dy, lddy, codes, scales, t, n, k, add,
                                                          stride, s);
        if (p.side == 128)
            return launch_wgrad<T, 128, 128, 64, 64, 64>(p, to, ld, to_db, (const T*)dy, lddy, codes, scales, t, n, k, add,
                                                         stride, s);
        return launch_wgrad<T, 64, 64, 32, 32, 64>(p, to, ld, to_db, (const T*)dy, lddy, codes, scales, t, n, k, add,
                                                   stride, s);
    }));
    if (!split) return NKMX_OK;
    return launch(join_parts_kernel, dim3((uint32_t)join_blocks), 256, s, dw, lddw, db, part, (uint32_t)p.parts, p.part_floats,
                  (uint32_t)n, (uint32_t)k, p.ldp, accumulate ? 1u : 0u);
}

}  // extern "C"
