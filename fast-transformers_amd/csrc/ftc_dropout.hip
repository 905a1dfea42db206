// The dropout behind a block, with the block's bias, activation and residual in the same pass over the rows, and its gradients
// (include/ftc_causal_product.h).
//
//   x_i = residual_i + keep_i act(z_i) / (1 - p),   z_i = block_i + bias,   keep_i = word_i >= p 2^32
//   grad_block_i = keep_i act'(z_i) grad_x_i / (1 - p),   grad_bias = its sums over the rows,   grad_residual = grad_x
//
// No mask is stored: word_i comes from a generator that is a function of i, the value's number among the rows' values, one row
// after the other, wherever they lie.  It is Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2,
// 3; 2011): ten rounds on a counter of four words, (i / 4, offset), with the seed as the key,
//
//   c <- (high(m1 c2) ^ c1 ^ k0, low(m1 c2), high(m0 c0) ^ c3 ^ k1, low(m0 c0)),   k0 += w0, k1 += w1
//
// whose four words are those of values 4 (i / 4) to 4 (i / 4) + 3.  A value has a word of 32 bits: p is a multiple of 2^-32, the nearest
// one, and the factor belongs to that one.
//
// A lane takes eight values of a row at a time; the last eight of a row whose width is no multiple of eight overlap those before,
// both lanes write the same.  All arithmetic is fp32, results are rounded once.  The sums for the bias: a workgroup walks rows with
// a lane's columns staying the same, and leaves them in the workspace for a second kernel, which adds them up in a fixed order.
//
// What bounds it: memory, for 40960 x 512 of fp32 onto a stream 48 us (252 MB, 5.2 TB/s) and back 32 (168 MB, 5.2 TB/s); with gelu the vector
// unit as well, 16384 x 8192 of bf16 147 to 152 us (537 MB, 3.6 TB/s) and back 176 (805 MB and 17 of sums, 4.7 TB/s), then 6 to add them up.  Without
// the generator, p = 0, the former is 8 to 12 % faster.
#include <algorithm>

#include "ftc_norm_kernel.h"

namespace ftc {
namespace dropout {
namespace {

using norm::any_u32x4;
using norm::kLot;
using norm::Rows;
using norm::u32x4;

constexpr int kThreads = 256;
// Lots of a lane that are on their way at a time.  Forward and backward, us, with one, two and four: 16384 x 8192 (bf16, bias, gelu) 336, 329, 336; 5411 x
// 1001 (bf16 onto fp32, bias, relu) 29.8, 30.1, 32.8; 40960 x 512 (fp32) 78, 78.5, 82.5.
constexpr int kAtOnce = 2;
constexpr int64_t kMostWidth = 1 << 18;
constexpr uint32_t kAll = 1 << 16;  // of the parts that p is counted in, each of 2^16 smaller ones

struct Args {
    Rows block, residual, x, grad_x, grad_block;
    const void *bias;
    int32_t bias_dtype, activation;
    int64_t rows;
    int32_t D, lots;      // lots: of a row
    uint32_t magic;       // n / lots = high(n magic), n up to lots + 2^10; 0: one lot
    uint32_t gone;        // p 2^32 - 1, the largest word of a value that is dropped (0 where none is)
    int32_t drops;        // whether any is
    float factor;         // 1 / (1 - p), or 0
    uint32_t seed[2], offset[2];
    const int64_t *seeds;  // seed and offset on the device, or null
    float *sums;           // for the bias: [part][D]
    int32_t across, parts; // lanes side by side, workgroups that walk the same columns
};

struct Lot {
    float x[kLot];
};
template <typename T>
struct Raw;
template <>
struct Raw<float> {
    u32x4 a, b;
};
template <>
struct Raw<uint16_t> {
    u32x4 a;
};
// (addresses of odd rows are anything that the type allows)
template <bool SHORT>
__device__ __forceinline__ void request(const float *from, int count, Raw<float> &r) {
    if (!SHORT) {
        r.a = ((const any_u32x4 *)from)[0], r.b = ((const any_u32x4 *)from)[1];
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            r.a[i] = i < count ? __float_as_uint(from[i]) : 0u;
            r.b[i] = 4 + i < count ? __float_as_uint(from[4 + i]) : 0u;
        }
    }
}
template <bool SHORT>
__device__ __forceinline__ void request(const uint16_t *from, int count, Raw<uint16_t> &r) {
    if (!SHORT) {
        r.a = *(const any_u32x4 *)from;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            r.a[i] = (2 * i < count ? (uint32_t)from[2 * i] : 0u) | (2 * i + 1 < count ? (uint32_t)from[2 * i + 1] : 0u) << 16;
    }
}
__device__ __forceinline__ Lot widen(const Raw<float> &r) {
    Lot l;
#pragma unroll
    for (int i = 0; i < 4; i++) l.x[i] = __uint_as_float(r.a[i]), l.x[4 + i] = __uint_as_float(r.b[i]);
    return l;
}
__device__ __forceinline__ Lot widen(const Raw<uint16_t> &r) {
    Lot l;
#pragma unroll
    for (int i = 0; i < 4; i++) l.x[2 * i] = __uint_as_float(r.a[i] << 16), l.x[2 * i + 1] = __uint_as_float(r.a[i] & 0xffff0000u);
    return l;
}
template <bool SHORT>
__device__ __forceinline__ void store(float *to, int count, const Lot &l) {
    if (!SHORT) {
#pragma unroll
        for (int h = 0; h < 2; h++)
            ((any_u32x4 *)to)[h] = u32x4{__float_as_uint(l.x[4 * h]), __float_as_uint(l.x[4 * h + 1]), __float_as_uint(l.x[4 * h + 2]),
                                         __float_as_uint(l.x[4 * h + 3])};
    } else {
#pragma unroll
        for (int i = 0; i < kLot; i++)
            if (i < count) to[i] = l.x[i];
    }
}
template <bool SHORT>
__device__ __forceinline__ void store(uint16_t *to, int count, const Lot &l) {
    if (!SHORT) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; i++)
            r[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{l.x[2 * i], l.x[2 * i + 1]}, bf16x2));
        *(any_u32x4 *)to = r;
    } else {
#pragma unroll
        for (int i = 0; i < kLot; i++)
            if (i < count) to[i] = f32_to_bf16(l.x[i]);
    }
}
template <bool SHORT>
__device__ __forceinline__ Lot load_bias(const Args &p, int col) {
    Lot l;
    if (!p.bias) {
#pragma unroll
        for (int i = 0; i < kLot; i++) l.x[i] = 0.f;
        return l;
    }
    const int count = SHORT ? p.D : kLot;
    if (p.bias_dtype == FTC_F32) {
        Raw<float> r;
        request<SHORT>((const float *)p.bias + col, count, r);
        return widen(r);
    }
    Raw<uint16_t> r;
    request<SHORT>((const uint16_t *)p.bias + col, count, r);
    return widen(r);
}

struct Place {
    int64_t row;
    int col;
};
// ---- the generator ----
struct Key {
    uint32_t k0, k1, o0, o1;
};
__device__ __forceinline__ Key key_of(const Args &p) {
    if (!p.seeds) return Key{p.seed[0], p.seed[1], p.offset[0], p.offset[1]};
    const uint64_t s = (uint64_t)p.seeds[0], o = (uint64_t)p.seeds[1];
    return Key{(uint32_t)s, (uint32_t)(s >> 32), (uint32_t)o, (uint32_t)(o >> 32)};
}
__device__ __forceinline__ u32x4 philox(uint64_t number, Key k) {
    uint32_t c0 = (uint32_t)number, c1 = (uint32_t)(number >> 32), c2 = k.o0, c3 = k.o1;
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k.k0, c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k.k1, c3 = (uint32_t)a;
        k.k0 += 0x9E3779B9u, k.k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1, c2, c3};
}
// The words of eight values from number `at` on, or the largest ones where nothing is dropped.  WHOLE: at is a multiple of four.
struct Words {
    uint32_t w[kLot];
};
template <bool WHOLE>
__device__ __forceinline__ Words words(const Args &p, const Place &place, const Key &k) {
    Words r;
    if (!p.drops) {  // (as in evaluation: no generator)
#pragma unroll
        for (int i = 0; i < kLot; i++) r.w[i] = ~0u;
        return r;
    }
    const uint64_t at = (uint64_t)(place.row * p.D + place.col);
    constexpr int kCounters = WHOLE ? 2 : 3;
    uint32_t w[4 * kCounters];
#pragma unroll
    for (int j = 0; j < kCounters; j++) {
        const u32x4 four = philox((at >> 2) + j, k);
#pragma unroll
        for (int i = 0; i < 4; i++) w[4 * j + i] = four[i];
    }
    if constexpr (!WHOLE) {
        const bool two = at & 2, one = at & 1;
        auto pick = [](bool other, uint32_t a, uint32_t b) { return other ? a : b; };
#pragma unroll
        for (int i = 0; i < kLot + 1; i++) w[i] = pick(two, w[i + 2], w[i]);
#pragma unroll
        for (int i = 0; i < kLot; i++) w[i] = pick(one, w[i + 1], w[i]);
    }
#pragma unroll
    for (int i = 0; i < kLot; i++) r.w[i] = w[i];
    return r;
}

// ---- activations ----
// The complement of the normal distribution, 1 - Phi(|z|): t P(t) e^{-x^2}, t = 1 / (1 + c x), x = |z| / sqrt 2, whose exponential serves for
// the density as well.  P was fitted for the least largest error relative to the value (x up to 14), so that the tail keeps its bits, which 1 + erf
// does not (fp32: 4 % at -5, nothing left at -5.5).  For results of fp32 of degree 9 to 4.5e-9 (its roundings in 32 bits come to 3.8e-7 at most, 7.5e-8
// in the mean); for gradients of bf16, which are added up in 32 bits for the bias, of degree 7 to 1.6e-7; for results of bf16 of degree 5 to 6.1e-6, a
// six hundredth of what rounding a result to bf16 may cost.  (16384 x 8192, fp32, with a bias, forward and with its backward: 239 and 524 us; 255 and 545
// with 1 + erf, 294 and 609 with erfc.)
template <int N>
__device__ __forceinline__ float behind(float z, float e, const float (&p)[N], float c) {
    const float t = __builtin_amdgcn_rcpf(fmaf(c, fabsf(z) * 0.70710678f, 1.f));
    float poly = p[N - 1];
#pragma unroll
    for (int i = N - 2; i >= 0; i--) poly = fmaf(poly, t, p[i]);
    return 0.5f * poly * t * e;
}
// Phi(z) and its density
template <bool FAST, bool SLOPE>
__device__ __forceinline__ float normal(float z, float &density) {
    const float e = __builtin_amdgcn_exp2f(z * z * -0.72134752f);
    density = 0.39894228f * e;
    constexpr float kSlope[] = {0.246796984f, 0.24770522f, 0.214494871f, 0.222751164f, -0.035136425f, 0.317385559f, -0.285824239f, 0.0718269597f},
                    kValue[] = {0.249892868f, 0.245066311f, 0.258995474f, 0.0543220965f, 0.335150677f, -0.143433497f};
    constexpr float kFull[] = {0.190403491f,  0.190687627f,  0.176482618f, 0.17770642f,   0.0470097065f,
                               0.303873807f, -0.316098958f, 0.435148358f, -0.256638408f, 0.0514253378f};
    const float half = !FAST ? behind(z, e, kFull, 0.3375f) : SLOPE ? behind(z, e, kSlope, 0.4375f) : behind(z, e, kValue, 0.4425f);
    return z < 0.f ? half : 1.f - half;
}
// 1 / (1 + e^{-z}), and what it lacks to one, from e^{-|z|}: neither is lost where the other is next to one
template <bool FAST>
__device__ __forceinline__ float logistic(float z, float &rest) {
    const float e = FAST ? __builtin_amdgcn_exp2f(fabsf(z) * -1.44269504f) : expf(-fabsf(z));
    const float r = FAST ? __builtin_amdgcn_rcpf(1.f + e) : 1.f / (1.f + e), other = e * r;
    rest = z < 0.f ? r : other;
    return z < 0.f ? other : r;
}
template <bool FAST>
__device__ __forceinline__ void activate(Lot &z, int activation) {
    if (activation == FTC_ACTIVATION_RELU) {
#pragma unroll
        for (int i = 0; i < kLot; i++) z.x[i] = z.x[i] <= 0.f ? 0.f : z.x[i];  // (NaN stays)
    } else if (activation == FTC_ACTIVATION_GELU) {
#pragma unroll
        for (int i = 0; i < kLot; i++) {
            float density;
            z.x[i] *= normal<FAST, false>(z.x[i], density);
        }
    } else if (activation == FTC_ACTIVATION_SILU) {
#pragma unroll
        for (int i = 0; i < kLot; i++) {
            float rest;
            z.x[i] *= logistic<FAST>(z.x[i], rest);
        }
    }
}
// their slopes, of which there are none where nothing is activated
template <bool FAST>
__device__ __forceinline__ void slopes(Lot &z, int activation) {
    if (activation == FTC_ACTIVATION_RELU) {
#pragma unroll
        for (int i = 0; i < kLot; i++) z.x[i] = z.x[i] <= 0.f ? 0.f : 1.f;  // (NaN passes it on, as it stays above)
    } else if (activation == FTC_ACTIVATION_GELU) {
#pragma unroll
        for (int i = 0; i < kLot; i++) {
            float density;
            const float phi = normal<FAST, true>(z.x[i], density);
            z.x[i] = fmaf(z.x[i], density, phi);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kLot; i++) {
            float rest;
            const float s = logistic<FAST>(z.x[i], rest);
            z.x[i] = s * (1.f + z.x[i] * rest);
        }
    }
}

// the lane's u-th lot of its workgroup's
__device__ __forceinline__ Place place_of(const Args &p, int64_t row0, uint32_t lot0, int u) {
    const uint32_t n = lot0 + threadIdx.x + kThreads * u;
    const uint32_t row = p.magic ? __umulhi(n, p.magic) : n;
    return Place{row0 + row, min((int)(n - row * (uint32_t)p.lots) * kLot, max(p.D - kLot, 0))};
}

// One lot's result
template <bool WHOLE, bool SHORT, bool FAST>
__device__ __forceinline__ void lot_forward(const Args &p, const Place &at, const Key &key, Lot &z, const Lot &bias, const Lot &onto) {
    const Words word = words<WHOLE>(p, at, key);
#pragma unroll
    for (int i = 0; i < kLot; i++) z.x[i] += bias.x[i];
    activate<FAST>(z, p.activation);
#pragma unroll
    for (int i = 0; i < kLot; i++) z.x[i] = (word.w[i] > p.gone ? z.x[i] * p.factor : 0.f) + onto.x[i];
}

// T: the block's type, X: that of x.  WHOLE: widths are multiples of four, SHORT: rows of fewer than eight.
template <typename T, typename X, bool WHOLE, bool SHORT>
__global__ __launch_bounds__(kThreads) void dropout_kernel(Args p) {
    const int64_t first = (int64_t)blockIdx.x * (kThreads * kAtOnce), row0 = first / p.lots;
    const uint32_t lot0 = (uint32_t)(first - row0 * p.lots);
    const Key key = key_of(p);
    const int count = SHORT ? p.D : kLot;
    Raw<T> block[kAtOnce];
    Raw<X> residual[kAtOnce];
    Place at[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) {
        at[u] = place_of(p, row0, lot0, u);
        if (at[u].row >= p.rows) continue;
        request<SHORT>((const T *)p.block.ptr + at[u].row * p.block.stride + at[u].col, count, block[u]);
        if (p.residual.ptr) request<SHORT>((const X *)p.residual.ptr + at[u].row * p.residual.stride + at[u].col, count, residual[u]);
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) {
        if (at[u].row >= p.rows) continue;
        Lot z = widen(block[u]);
        lot_forward<WHOLE, SHORT, sizeof(X) == 2>(p, at[u], key, z, Lot{}, p.residual.ptr ? widen(residual[u]) : Lot{});
        store<SHORT>((X *)p.x.ptr + at[u].row * p.x.stride + at[u].col, count, z);
    }
}

// ... with a bias: a workgroup's lanes keep their columns and walk the rows.  (us, and with the bias loaded with every lot: 5411 x 1001 13.7, 14.9;
// 16384 x 8192 147, 148; 20000 x 768 25.7, 22.7.)
template <typename T, typename X, bool WHOLE, bool SHORT>
__global__ __launch_bounds__(kThreads) void dropout_bias_kernel(Args p) {
    const int across = p.across, teams = kThreads / across, lane = threadIdx.x % across, team = threadIdx.x / across;
    const int lot = (int)blockIdx.y * across + lane, col = min(lot * kLot, max(p.D - kLot, 0));
    const int count = SHORT ? p.D : kLot;
    if (lot >= p.lots) return;
    const Key key = key_of(p);
    const Lot bias = load_bias<SHORT>(p, col);
    const int64_t step = (int64_t)p.parts * teams;
    for (int64_t row = (int64_t)blockIdx.x * teams + team; row < p.rows; row += kAtOnce * step) {
        Raw<T> block[kAtOnce];
        Raw<X> residual[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            const int64_t r = row + u * step;
            if (r >= p.rows) continue;
            request<SHORT>((const T *)p.block.ptr + r * p.block.stride + col, count, block[u]);
            if (p.residual.ptr) request<SHORT>((const X *)p.residual.ptr + r * p.residual.stride + col, count, residual[u]);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            const Place at{row + u * step, col};
            if (at.row >= p.rows) continue;
            Lot z = widen(block[u]);
            lot_forward<WHOLE, SHORT, sizeof(X) == 2>(p, at, key, z, bias, p.residual.ptr ? widen(residual[u]) : Lot{});
            store<SHORT>((X *)p.x.ptr + at.row * p.x.stride + col, count, z);
        }
    }
}

// One lot's gradient
template <bool WHOLE, bool SHORT, bool FAST>
__device__ __forceinline__ void lot_back(const Args &p, const Place &at, const Key &key, Lot z, const Lot &bias, Lot &grad) {
    const Words word = words<WHOLE>(p, at, key);
    if (p.activation != FTC_ACTIVATION_NONE) {
#pragma unroll
        for (int i = 0; i < kLot; i++) z.x[i] += bias.x[i];
        slopes<FAST>(z, p.activation);
#pragma unroll
        for (int i = 0; i < kLot; i++) grad.x[i] *= z.x[i];
    }
#pragma unroll
    for (int i = 0; i < kLot; i++) grad.x[i] = word.w[i] > p.gone ? grad.x[i] * p.factor : 0.f;
}

template <typename T, typename X, bool WHOLE, bool SHORT>
__global__ __launch_bounds__(kThreads) void dropout_back_kernel(Args p) {
    const int64_t first = (int64_t)blockIdx.x * (kThreads * kAtOnce), row0 = first / p.lots;
    const uint32_t lot0 = (uint32_t)(first - row0 * p.lots);
    const Key key = key_of(p);
    const int count = SHORT ? p.D : kLot;
    Raw<T> block[kAtOnce];
    Raw<X> grad_x[kAtOnce];
    Place at[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) {
        at[u] = place_of(p, row0, lot0, u);
        if (at[u].row >= p.rows) continue;
        request<SHORT>((const X *)p.grad_x.ptr + at[u].row * p.grad_x.stride + at[u].col, count, grad_x[u]);
        if (p.activation != FTC_ACTIVATION_NONE)
            request<SHORT>((const T *)p.block.ptr + at[u].row * p.block.stride + at[u].col, count, block[u]);
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; u++) {
        if (at[u].row >= p.rows) continue;
        Lot grad = widen(grad_x[u]), z = Lot{}, bias = Lot{};
        if (p.activation != FTC_ACTIVATION_NONE) z = widen(block[u]), bias = load_bias<SHORT>(p, at[u].col);
        lot_back<WHOLE, SHORT, sizeof(T) == 2>(p, at[u], key, z, bias, grad);
        store<SHORT>((T *)p.grad_block.ptr + at[u].row * p.grad_block.stride + at[u].col, count, grad);
    }
}

// ... with the sums for the bias: a workgroup's lanes keep their columns
template <typename T, typename X, bool WHOLE, bool SHORT>
__global__ __launch_bounds__(kThreads) void dropout_back_bias_kernel(Args p) {
    __shared__ float mem[kThreads * kLot];
    const int across = p.across, teams = kThreads / across, lane = threadIdx.x % across, team = threadIdx.x / across;
    const int lot = (int)blockIdx.y * across + lane, col = min(lot * kLot, max(p.D - kLot, 0));
    const int count = SHORT ? p.D : kLot;
    const Key key = key_of(p);
    Lot sum = Lot{};
    if (lot < p.lots) {
        const Lot bias = load_bias<SHORT>(p, col);
        const int64_t step = (int64_t)p.parts * teams;
        for (int64_t row = (int64_t)blockIdx.x * teams + team; row < p.rows; row += kAtOnce * step) {
            Raw<T> block[kAtOnce];
            Raw<X> grad_x[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; u++) {
                const int64_t r = row + u * step;
                if (r >= p.rows) continue;
                request<SHORT>((const X *)p.grad_x.ptr + r * p.grad_x.stride + col, count, grad_x[u]);
                if (p.activation != FTC_ACTIVATION_NONE)
                    request<SHORT>((const T *)p.block.ptr + r * p.block.stride + col, count, block[u]);
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; u++) {
                const Place at{row + u * step, col};
                if (at.row >= p.rows) continue;
                Lot grad = widen(grad_x[u]), z = p.activation != FTC_ACTIVATION_NONE ? widen(block[u]) : Lot{};
                lot_back<WHOLE, SHORT, sizeof(T) == 2>(p, at, key, z, bias, grad);
                if (p.grad_block.ptr) store<SHORT>((T *)p.grad_block.ptr + at.row * p.grad_block.stride + col, count, grad);
#pragma unroll
                for (int i = 0; i < kLot; i++) sum.x[i] += grad.x[i];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kLot; i++) mem[threadIdx.x * kLot + i] = sum.x[i];
    __syncthreads();
    if (team != 0 || lot >= p.lots) return;
    for (int t = 1; t < teams; t++)
#pragma unroll
        for (int i = 0; i < kLot; i++) sum.x[i] += mem[(t * across + lane) * kLot + i];
#pragma unroll
    for (int i = 0; i < kLot; i++)  // (columns that the lot before has as well are its)
        if (i < count && col + i >= lot * kLot) p.sums[(int64_t)blockIdx.x * p.D + col + i] = sum.x[i];
}

// ---- host ----
int read_rows(const ftc_rows *r, const char *name, bool wanted, Rows *to) {
    *to = Rows{};
    if (!r || !r->ptr) return wanted ? fail(FTC_ERR_INVALID, "%s is null", name) : FTC_OK;
    if (r->dtype != FTC_F32 && r->dtype != FTC_BF16)
        return fail(FTC_ERR_INVALID, "%s has dtype code %d, expected FTC_F32 or FTC_BF16", name, (int)r->dtype);
    *to = Rows{r->ptr, r->stride, r->dtype};
    return FTC_OK;
}
int read_call(const ftc_residual_dropout_call *c, bool back, Args *p) {
    if (!c) return fail(FTC_ERR_INVALID, "the call is null");
    if (c->rows < 0 || c->width < 1) return fail(FTC_ERR_INVALID, "rows of at least one value are taken, got %lld of %lld",
                                                 (long long)c->rows, (long long)c->width);
    // (a launch has fewer than 2^32 lanes, of two lots each)
    if (c->width > kMostWidth || c->rows > ((int64_t)1 << 32) / ((c->width + kLot - 1) / kLot))
        return fail(FTC_ERR_UNSUPPORTED, "rows of up to %lld values are supported, 2^35 values in all", (long long)kMostWidth);
    if (c->activation < FTC_ACTIVATION_NONE || c->activation > FTC_ACTIVATION_SILU)
        return fail(FTC_ERR_INVALID, "the activation has code %d", (int)c->activation);
    if (c->dropped > kAll || c->dropped_rest >= kAll || (c->dropped == kAll && c->dropped_rest))
        return fail(FTC_ERR_INVALID, "%u parts in 65536 and %u in 2^32 cannot be dropped", (unsigned)c->dropped, (unsigned)c->dropped_rest);
    if (c->bias && c->bias_dtype != FTC_F32 && c->bias_dtype != FTC_BF16)
        return fail(FTC_ERR_INVALID, "the bias has dtype code %d", (int)c->bias_dtype);
    const bool reads = !back || c->activation != FTC_ACTIVATION_NONE;
    if (int rc = read_rows(&c->block, "block", reads && c->rows > 0, &p->block)) return rc;
    if (int rc = read_rows(&c->residual, "residual", false, &p->residual)) return rc;
    p->bias = c->bias, p->bias_dtype = c->bias_dtype, p->activation = c->activation;
    p->rows = c->rows, p->D = (int32_t)c->width, p->lots = (p->D + kLot - 1) / kLot;
    p->magic = p->lots == 1 ? 0 : (uint32_t)(((uint64_t)1 << 32) / (uint32_t)p->lots + 1);
    const uint64_t all = (uint64_t)kAll * kAll, border = (uint64_t)c->dropped * kAll + c->dropped_rest;
    p->drops = border > 0, p->gone = border > 0 ? (uint32_t)(border - 1) : 0;
    p->factor = border == all ? 0.f : (float)((double)all / (double)(all - border));
    p->seed[0] = (uint32_t)c->seed, p->seed[1] = (uint32_t)(c->seed >> 32);
    p->offset[0] = (uint32_t)c->offset, p->offset[1] = (uint32_t)(c->offset >> 32);
    p->seeds = c->seeds;
    return FTC_OK;
}
// Workgroups that walk rows: 2048, eight a compute unit, but not so many that a team has fewer than four rows (each leaves a row of sums,
// which are added up later), down to 512.  Measured, forward and backward, us, by the least number of rows, 1, 2, 4, 8: 5411 x 1001 (bf16 onto fp32,
// relu) 35.3, 33.5, 30.1, 31.4; of bf16 with gelu 1000 x 4096 34.2, 27.6, 24.9, 25.0; 20000 x 768 60.5, 61.0, 60.6, 61.1; 16384 x 8192 (512 parts of
// four columns of workgroups) 328 to 337 whichever.
void plan_walk(Args *p) {
    p->across = 1;
    while (p->across < p->lots && p->across < kThreads) p->across *= 2;
    const int64_t columns = (p->lots + p->across - 1) / p->across, teams = kThreads / p->across;
    const int64_t most = (p->rows + teams - 1) / teams, groups = std::clamp<int64_t>(columns * most / 4, 512, 2048);
    p->parts = (int32_t)std::max<int64_t>(1, std::min(most, groups / columns));
}
int launched(const char *name) {
    note_kernel(name);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FTC_OK : fail(FTC_ERR_HIP, "%s: %s", name, hipGetErrorString(e));
}

template <typename T, typename X, bool WHOLE, bool SHORT>
void run(const Args &p, int what, hipStream_t stream) {
    const int64_t per = kThreads * kAtOnce, groups = (p.rows * p.lots + per - 1) / per;
    if (what == 0) dropout_kernel<T, X, WHOLE, SHORT><<<dim3((uint32_t)groups), kThreads, 0, stream>>>(p);
    else if (what == 1) dropout_back_kernel<T, X, WHOLE, SHORT><<<dim3((uint32_t)groups), kThreads, 0, stream>>>(p);
    else {
        const dim3 grid((uint32_t)p.parts, (uint32_t)((p.lots + p.across - 1) / p.across));
        if (what == 2) dropout_back_bias_kernel<T, X, WHOLE, SHORT><<<grid, kThreads, 0, stream>>>(p);
        else dropout_bias_kernel<T, X, WHOLE, SHORT><<<grid, kThreads, 0, stream>>>(p);
    }
}
// what: 0 forward, 1 the gradient of the block, 2 that of the bias as well, 3 forward with a bias
void dispatch(const Args &p, bool block_f32, bool x_f32, int what, hipStream_t stream) {
    auto widths = [&](auto t, auto x) {
        using T = decltype(t);
        using X = decltype(x);
        if (p.D < kLot) run<T, X, false, true>(p, what, stream);
        else if (p.D % 4 == 0) run<T, X, true, false>(p, what, stream);
        else run<T, X, false, false>(p, what, stream);
    };
    if (block_f32) x_f32 ? widths(float(), float()) : widths(float(), uint16_t());
    else x_f32 ? widths(uint16_t(), float()) : widths(uint16_t(), uint16_t());
}

}  // namespace
}  // namespace dropout
}  // namespace ftc

using namespace ftc;
using namespace ftc::dropout;

extern "C" {

int ftc_residual_dropout(const ftc_residual_dropout_call *call, const ftc_rows *x, void *stream) {
    Args p = {};
    if (int rc = read_call(call, false, &p)) return rc;
    if (int rc = read_rows(x, "x", p.rows > 0, &p.x)) return rc;
    if (p.rows == 0) return FTC_OK;
    if (p.residual.ptr && p.residual.dtype != p.x.dtype) return fail(FTC_ERR_INVALID, "x and the residual must have one dtype");
    if (p.bias) plan_walk(&p);
    dispatch(p, p.block.dtype == FTC_F32, p.x.dtype == FTC_F32, p.bias ? 3 : 0, (hipStream_t)stream);
    return launched(p.bias ? "dropout_bias_kernel" : "dropout_kernel");
}

int64_t ftc_residual_dropout_backward_workspace_bytes(const ftc_residual_dropout_call *call) {
    Args p = {};
    if (int rc = read_call(call, true, &p)) return rc;
    if (p.rows == 0) return 0;
    plan_walk(&p);
    return 4 * (int64_t)p.parts * p.D;
}

int ftc_residual_dropout_backward(const ftc_residual_dropout_call *call, const ftc_rows *grad_x, const ftc_rows *grad_block,
                                  void *grad_bias, void *workspace, size_t workspace_bytes, void *stream) {
    Args p = {};
    if (int rc = read_call(call, true, &p)) return rc;
    if (int rc = read_rows(grad_x, "grad_x", p.rows > 0, &p.grad_x)) return rc;
    if (int rc = read_rows(grad_block, "grad_block", false, &p.grad_block)) return rc;
    if (grad_bias && !p.bias) return fail(FTC_ERR_INVALID, "grad_bias is given without a bias");
    if (p.rows == 0 || (!grad_bias && !p.grad_block.ptr)) return FTC_OK;
    if (p.block.ptr && p.grad_block.ptr && p.block.dtype != p.grad_block.dtype)
        return fail(FTC_ERR_INVALID, "grad_block must have the block's dtype");
    const bool block_f32 = (p.block.ptr ? p.block.dtype : p.grad_block.ptr ? p.grad_block.dtype : p.grad_x.dtype) == FTC_F32;
    if (!grad_bias) {
        dispatch(p, block_f32, p.grad_x.dtype == FTC_F32, 1, (hipStream_t)stream);
        return launched("dropout_back_kernel");
    }
    plan_walk(&p);
    const int64_t need = 4 * (int64_t)p.parts * p.D;
    if (!workspace || (int64_t)workspace_bytes < need)
        return fail(FTC_ERR_WORKSPACE, "ftc_residual_dropout_backward needs %lld bytes", (long long)need);
    if ((uintptr_t)workspace & 255) return fail(FTC_ERR_WORKSPACE, "the workspace must be 256-byte aligned");
    p.sums = (float *)workspace;
    dispatch(p, block_f32, p.grad_x.dtype == FTC_F32, 2, (hipStream_t)stream);
    norm::FoldArgs f = {};
    f.D = p.D, f.folds = 1;
    f.fold[0] = norm::Fold{p.sums, grad_bias, 0, 0, p.bias_dtype, 1, p.parts, p.D};
    norm::fold_rows(f, 1, (hipStream_t)stream);
    return launched("dropout_back_bias_kernel");
}

}  // extern "C"
