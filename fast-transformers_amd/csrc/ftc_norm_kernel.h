// The norms around a block, its gate and residual in one pass over the rows, and their gradients.
//
//   n = norm_after(block),  y = n w_a + b_a,  x = residual + scale act(gate) y,  h = norm_before(x) w_b + b_b
//   norm: (r - mean) / sqrt(variance + eps), or r / sqrt(mean of squares + eps), or r itself
//
// Backward, with x^ the normalised x and the norms' statistics from the forward:
//   dx = grad_x + rstd (w_b grad_h - [mean of it] - x^ mean(w_b grad_h x^)),   grad_residual = dx
//   dy = scale act(gate) dx,   grad_gate = scale act'(gate) y dx,   grad_block = the same of the first norm, from dy
//   gradients of w_b, b_b, w_a, b_a: sums over the rows of grad_h x^, grad_h, dy n, dy
//
// What bounds it is memory: every row is read once and written once, held in registers in between (x is made again in
// the backward from the same rows that it has to read anyway: a stored x in 16 bits would spoil the gradients of w_b).
// A team of 16 to 1024 lanes takes a row, eight values a lane at a time; the workgroup walks its rows and keeps the
// sums for the parameters in registers, leaves them in the workspace, and a second kernel adds them up in a fixed
// order.  A gate that several rows share is summed the same way: a workgroup's rows all belong to one of its rows.
// All arithmetic is fp32; results are rounded once.
//
// Measured, forward | backward, of all bytes read and written: 40960 x 512, fp32, 76 us | 119 us, 4.4 | 4.2 TB/s; 16384 x 4096, bf16 beside
// an fp32 stream, 180 | 390, 5.2 | 3.8; 524288 x 128, bf16, 97 | 147, 4.1 | 4.6 (a copy: 5.1).  The backward of rows above
// 2048 has one workgroup a compute unit, by its registers: held to 128 of them it spills (440 us), and with the next
// row requested ahead it takes 430.
#pragma once
#include <initializer_list>

#include "ftc_common.h"

namespace ftc {
namespace norm {

constexpr int kLot = 8;  // values of a row that a lane takes at a time

struct Params {
    const void *weight, *bias;
    int32_t kind, weight_dtype, bias_dtype;  // kind: enum ftc_norm_kind
};
struct Rows {
    void *ptr;
    int64_t stride;
    int32_t dtype;
};
struct Args {
    Rows block, residual, gate, x, h, grad_x, grad_h, grad_block, grad_residual, grad_gate;
    Params after, before;
    float *stats;        // four floats a row: mean and 1 / deviation of the first norm and of the second
    float *sums;         // partial sums for the parameters, [workgroup][kSums][D]
    float *gate_sums;    // ... and for a shared gate, [gate row][part][D]
    int64_t rows, gate_rows, every;  // every: rows that have the same gate row
    int64_t segment;                 // rows that the backward sums together: `every` of a shared gate, else all
    int32_t D, parts, activation, shared;  // parts: workgroups per segment; shared: several rows have one gate row
    float scale, eps;
};
enum { kAfterWeight, kAfterBias, kBeforeWeight, kBeforeBias, kSums };

struct Lot {
    float x[kLot];
};
// 16 bytes at any address that the values' type allows (rows of odd widths start there)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t any_u32x4 __attribute__((ext_vector_type(4), aligned(2), may_alias));

// A lot as it comes from memory: widening it where it is requested would wait for it.  TAIL: a row may end inside it
// (`left` values of it are there).  Then it is the row's last eight values that are read, in one access as well, and they are
// moved to their places when they are widened, with zeros behind: read one by one, which has to wait for them, rows of 1023
// bf16 values took 256 us forward and 735 back instead of 152 and 352 (60000 of them).  Rows of fewer than eight
// are read so all the same, and tails of those that leave no registers for the moves (MOVE; two lots a lane: 8190 values,
// 194 forward and 436 back, with the moves 235 and 532).
struct Raw {
    u32x4 a, b;
};
template <bool TAIL, bool MOVE>
__device__ __forceinline__ Raw request(const void *base, int dtype, int64_t at, int left, bool is_short) {
    Raw r;
    if (!TAIL || (MOVE ? !is_short : left >= kLot)) {
        if (TAIL && MOVE && left < kLot) at -= kLot - left;
        const char *const from = (const char *)base + at * (dtype == FTC_F32 ? 4 : 2);
        r.a = *(const any_u32x4 *)from;
        if (dtype == FTC_F32) r.b = *(const any_u32x4 *)(from + 16);
    } else {
        const char *const from = (const char *)base + at * (dtype == FTC_F32 ? 4 : 2);
        uint32_t x[kLot];
#pragma unroll
        for (int i = 0; i < kLot; i++)
            x[i] = i >= left ? 0u : dtype == FTC_F32 ? ((const uint32_t *)from)[i] : (uint32_t)((const uint16_t *)from)[i];
        if (dtype == FTC_F32) r.a = u32x4{x[0], x[1], x[2], x[3]}, r.b = u32x4{x[4], x[5], x[6], x[7]};
        else r.a = u32x4{x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16};
    }
    return r;
}
template <bool TAIL, bool MOVE>
__device__ __forceinline__ Lot widen(const Raw &r, int dtype, int left, bool is_short) {
    Lot x;
    if (dtype == FTC_F32) {
#pragma unroll
        for (int i = 0; i < 4; i++) x.x[i] = __uint_as_float(r.a[i]), x.x[4 + i] = __uint_as_float(r.b[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            x.x[2 * i] = __uint_as_float(r.a[i] << 16), x.x[2 * i + 1] = __uint_as_float(r.a[i] & 0xffff0000u);
    }
    if (TAIL && MOVE && left < kLot && !is_short) {
        const int by = kLot - left;
#pragma unroll
        for (int bit = 4; bit >= 1; bit /= 2)
            if (by & bit)
#pragma unroll
                for (int i = 0; i < kLot; i++) x.x[i] = i + bit < kLot ? x.x[(i + bit) % kLot] : 0.f;
    }
    return x;
}
template <bool TAIL>
__device__ __forceinline__ void store_lot(void *base, int dtype, int64_t at, int left, const Lot &r) {
    if (!TAIL || left >= kLot) {
        if (dtype == FTC_F32) {
            any_u32x4 *const to = (any_u32x4 *)((float *)base + at);
#pragma unroll
            for (int h = 0; h < 2; h++)
                to[h] = u32x4{__float_as_uint(r.x[4 * h]), __float_as_uint(r.x[4 * h + 1]), __float_as_uint(r.x[4 * h + 2]),
                              __float_as_uint(r.x[4 * h + 3])};
        } else {
            typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
            typedef float f32x2 __attribute__((ext_vector_type(2)));
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; i++)
                w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{r.x[2 * i], r.x[2 * i + 1]}, bf16x2));
            *(any_u32x4 *)((uint16_t *)base + at) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kLot; i++)
            if (i < left) store_from_f32(base, dtype, at + i, r.x[i]);
    }
}

// Sums over a team of LPR lanes, two at a time, in every lane; `turn` alternates between the two halves of `mem`
// so that one barrier is enough.
template <int LPR>
__device__ __forceinline__ void team_sum(float &a, float &b, float (*mem)[2][16], int &turn) {
#pragma unroll
    for (int d = 1; d < (LPR < 64 ? LPR : 64); d *= 2) a += __shfl_xor(a, d), b += __shfl_xor(b, d);
    if (LPR > 64) {
        constexpr int kWaves = LPR / 64;
        const int wave = threadIdx.x >> 6, first = wave / kWaves * kWaves;
        if ((threadIdx.x & 63) == 0) mem[turn][0][wave] = a, mem[turn][1][wave] = b;
        __syncthreads();
        a = 0.f, b = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) a += mem[turn][0][first + w], b += mem[turn][1][first + w];
        turn ^= 1;
    }
}

// The gate's factor and its slope.  s = 1 / (1 + exp(-g)) and 1 - s from the hardware's 2^x of the exponent's whole product
// (its rounding made good, since it is multiplied by the exponent) and its reciprocal: within 3 half steps, and 7.  Gates
// below -88.5 count as that (2^x would be infinite a little further): s is then under 2^-127, which the reciprocal gives as
// zero.  A NaN stays one.
__device__ __forceinline__ void activate(float g, int activation, float &value, float &slope) {
    if (activation == FTC_GATE_PLAIN) {
        value = g, slope = 1.f;
        return;
    }
    constexpr float kLog2e = 1.44269502f, kRest = 1.92596299e-8f;  // log2(e) in two floats
    const float low = __builtin_elementwise_maximum(g, -88.5f), x = __builtin_elementwise_minimum(low, 126.f);
    const float t = x * -kLog2e, lost = fmaf(x, -kRest, fmaf(x, -kLog2e, -t));
    const float two = __builtin_amdgcn_exp2f(t), e = fmaf(two, lost * 0.693147181f, two);
    const float s = __builtin_amdgcn_rcpf(1.f + e), rest = e * s;
    if (activation == FTC_GATE_SIGMOID) value = s, slope = s * rest;
    else value = low * s, slope = s * fmaf(x, rest, 1.f);
}

// One lot of a norm's weight and bias (from the caches: where they are used)
template <bool TAIL, bool MOVE>
__device__ __forceinline__ void params_lot(const Params &p, int col, int left, bool is_short, Lot &w, Lot &b) {
    if (p.weight) w = widen<TAIL, MOVE>(request<TAIL, MOVE>(p.weight, p.weight_dtype, col, left, is_short), p.weight_dtype, left, is_short);
    else
#pragma unroll
        for (int i = 0; i < kLot; i++) w.x[i] = 1.f;
    if (p.bias) b = widen<TAIL, MOVE>(request<TAIL, MOVE>(p.bias, p.bias_dtype, col, left, is_short), p.bias_dtype, left, is_short);
    else
#pragma unroll
        for (int i = 0; i < kLot; i++) b.x[i] = 0.f;
}
// The type of rows that the kernel is made for, or any
template <int DTYPE>
__device__ __forceinline__ int type_of(const Rows &r) {
    return DTYPE >= 0 ? DTYPE : r.dtype;
}

// LPR lanes take a row, NV lots each; THREADS / LPR rows at a time
// DB, DS: types of the block's rows (gate and h too) and of the stream's
template <int LPR, int NV, bool TAIL, int DB, int DS>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void residual_norm_kernel(Args p) {
    constexpr int kThreads = LPR > 256 ? LPR : 256, kTeams = kThreads / LPR;
    __shared__ float mem[2][2][16];
    const int team = threadIdx.x / LPR, lane = threadIdx.x % LPR;
    int turn = 0;
    const float per = 1.f / (float)p.D;
    constexpr bool MOVE = NV == 1;
    const bool is_short = p.D < kLot;
    auto column = [&](int v) { return kLot * (lane + LPR * v); };

    // Mean (layer norm) and 1 / deviation of the row in r
    auto statistics = [&](const Lot (&r)[NV], const Params &n, float &mean, float &rstd) {
        mean = 0.f, rstd = 1.f;
        if (n.kind == FTC_NORM_NONE) return;
        float none = 0.f;
        if (n.kind == FTC_NORM_LAYER) {
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int i = 0; i < kLot; i++) mean += r[v].x[i];  // (zeros past the row's end)
            team_sum<LPR>(mean, none, mem, turn);
            mean *= per;
        }
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int i = 0; i < kLot; i++)
                if (column(v) + (TAIL ? i : 0) < p.D) sum = fmaf(r[v].x[i] - mean, r[v].x[i] - mean, sum);
        team_sum<LPR>(sum, none, mem, turn);
        rstd = 1.f / sqrtf(sum * per + p.eps);
    };

    for (int64_t base = (int64_t)blockIdx.x * kTeams; base < p.rows; base += (int64_t)gridDim.x * kTeams) {
        const int64_t row = base + team, gate_row = p.every == 1 ? row : (uint32_t)row / (uint32_t)p.every;  // (fewer than 2^31)
        const bool live = row < p.rows;
        Raw block[NV], gate[NV], residual[NV];
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int col = column(v), left = p.D - col;
            if (!live || left <= 0) continue;
            block[v] = request<TAIL, MOVE>(p.block.ptr, type_of<DB>(p.block), row * p.block.stride + col, left, is_short);
            if (p.gate.ptr) gate[v] = request<TAIL, MOVE>(p.gate.ptr, type_of<DB>(p.gate), gate_row * p.gate.stride + col, left, is_short);
            if (p.residual.ptr)
                residual[v] = request<TAIL, MOVE>(p.residual.ptr, type_of<DS>(p.residual), row * p.residual.stride + col, left, is_short);
        }
        Lot r[NV];
#pragma unroll
        for (int v = 0; v < NV; v++) {
            if (live && column(v) < p.D) r[v] = widen<TAIL, MOVE>(block[v], type_of<DB>(p.block), p.D - column(v), is_short);
            else
#pragma unroll
                for (int i = 0; i < kLot; i++) r[v].x[i] = 0.f;
        }
        float mean_a, rstd_a, mean_b, rstd_b;
        statistics(r, p.after, mean_a, rstd_a);
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int col = column(v);
            if (!live || col >= p.D) continue;
            if (p.after.kind != FTC_NORM_NONE) {
                Lot w, b;
                params_lot<TAIL, MOVE>(p.after, col, p.D - col, is_short, w, b);
#pragma unroll
                for (int i = 0; i < kLot; i++) r[v].x[i] = fmaf((r[v].x[i] - mean_a) * rstd_a, w.x[i], b.x[i]);
            }
            if (p.gate.ptr) {
                const Lot g = widen<TAIL, MOVE>(gate[v], type_of<DB>(p.gate), p.D - column(v), is_short);
#pragma unroll
                for (int i = 0; i < kLot; i++) {
                    float value, slope;
                    activate(g.x[i], p.activation, value, slope);
                    r[v].x[i] *= value;
                }
            }
            if (p.residual.ptr) {
                const Lot d = widen<TAIL, MOVE>(residual[v], type_of<DS>(p.residual), p.D - column(v), is_short);
#pragma unroll
                for (int i = 0; i < kLot; i++) r[v].x[i] = fmaf(p.scale, r[v].x[i], d.x[i]);
            } else {
#pragma unroll
                for (int i = 0; i < kLot; i++) r[v].x[i] *= p.scale;
            }
            if (TAIL)
#pragma unroll
                for (int i = 0; i < kLot; i++) r[v].x[i] = col + i < p.D ? r[v].x[i] : 0.f;
            store_lot<TAIL>(p.x.ptr, type_of<DS>(p.x), row * p.x.stride + col, p.D - col, r[v]);
        }
        statistics(r, p.before, mean_b, rstd_b);
        if (p.h.ptr && live)
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int col = column(v);
                if (col >= p.D) continue;
                Lot w, b;
                params_lot<TAIL, MOVE>(p.before, col, p.D - col, is_short, w, b);
#pragma unroll
                for (int i = 0; i < kLot; i++) r[v].x[i] = fmaf((r[v].x[i] - mean_b) * rstd_b, w.x[i], b.x[i]);
                store_lot<TAIL>(p.h.ptr, type_of<DB>(p.h), row * p.h.stride + col, p.D - col, r[v]);
            }
        if (p.stats && live && lane == 0)
            *(float4 *)(p.stats + 4 * row) = make_float4(mean_a, rstd_a, mean_b, rstd_b);
    }
}

// FULL: a norm has a bias, or several rows have one gate row
template <int LPR, int NV, bool TAIL, int DB, int DS, bool FULL>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void residual_norm_backward_kernel(Args p) {
    constexpr int kThreads = LPR > 256 ? LPR : 256, kTeams = kThreads / LPR;
    __shared__ float mem[2][2][16];
    __shared__ float fold_mem[kTeams > 1 ? kTeams * LPR * kLot * NV : 1];
    const int team = threadIdx.x / LPR, lane = threadIdx.x % LPR;
    int turn = 0;
    const float per = 1.f / (float)p.D;
    constexpr bool MOVE = NV == 1;
    const bool is_short = p.D < kLot;
    auto column = [&](int v) { return kLot * (lane + LPR * v); };
    // the teams' sums to one row of floats
    auto leave = [&](auto &sum, float *to) {
        if (kTeams > 1) {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int i = 0; i < kLot; i++) fold_mem[(team * LPR * NV + lane * NV + v) * kLot + i] = sum[v].x[i];
            __syncthreads();
            if (team) return;
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int i = 0; i < kLot; i++) {
                    float s = sum[v].x[i];
#pragma unroll
                    for (int t = 1; t < kTeams; t++) s += fold_mem[(t * LPR * NV + lane * NV + v) * kLot + i];
                    sum[v].x[i] = s;
                }
        }
#pragma unroll
        for (int v = 0; v < NV; v++)
            if (column(v) < p.D) store_lot<TAIL>(to, FTC_F32, column(v), p.D - column(v), sum[v]);
    };

    Lot dwa[NV] = {}, dba[FULL ? NV : 1] = {}, dwb[NV] = {}, dbb[FULL ? NV : 1] = {};
    // segments of rows (one per gate row), the part of them that is this workgroup's
    const int part = blockIdx.x % p.parts;
    for (int64_t seg = blockIdx.x / p.parts; seg * p.segment < p.rows; seg += gridDim.x / p.parts) {
        const int64_t first = seg * p.segment, end = min(p.rows, first + p.segment);
        Lot dgate[FULL ? NV : 1] = {};
        for (int64_t base = first + (int64_t)part * kTeams; base < end; base += (int64_t)p.parts * kTeams) {
            const int64_t row = base + team, gate_row = FULL && p.shared ? seg : row;
            const bool live = row < end;
            float mean_a = 0.f, rstd_a = 1.f, mean_b = 0.f, rstd_b = 1.f;
            if (live && p.stats) {
                const float4 s = *(const float4 *)(p.stats + 4 * row);
                mean_a = s.x, rstd_a = s.y, mean_b = s.z, rstd_b = s.w;
            }
            Raw block_raw[NV], gate_raw[NV], residual_raw[NV], gh_raw[NV], gx_raw[NV];
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int col = column(v), left = p.D - col;
                if (!live || left <= 0) continue;
                block_raw[v] = request<TAIL, MOVE>(p.block.ptr, type_of<DB>(p.block), row * p.block.stride + col, left, is_short);
                if (p.gate.ptr) gate_raw[v] = request<TAIL, MOVE>(p.gate.ptr, type_of<DB>(p.gate), gate_row * p.gate.stride + col, left, is_short);
                if (p.before.kind != FTC_NORM_NONE) {
                    if (p.residual.ptr)
                        residual_raw[v] = request<TAIL, MOVE>(p.residual.ptr, type_of<DS>(p.residual), row * p.residual.stride + col, left, is_short);
                    if (p.grad_h.ptr) gh_raw[v] = request<TAIL, MOVE>(p.grad_h.ptr, type_of<DB>(p.grad_h), row * p.grad_h.stride + col, left, is_short);
                }
                if (p.grad_x.ptr) gx_raw[v] = request<TAIL, MOVE>(p.grad_x.ptr, type_of<DS>(p.grad_x), row * p.grad_x.stride + col, left, is_short);
            }
            Lot n[NV], dx[NV], gate[NV], xh[NV];
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int col = column(v), left = p.D - col;
#pragma unroll
                for (int i = 0; i < kLot; i++) n[v].x[i] = dx[v].x[i] = xh[v].x[i] = gate[v].x[i] = 0.f;
                if (!live || col >= p.D) continue;
                n[v] = widen<TAIL, MOVE>(block_raw[v], type_of<DB>(p.block), p.D - column(v), is_short);
                if (p.gate.ptr) gate[v] = widen<TAIL, MOVE>(gate_raw[v], type_of<DB>(p.gate), p.D - column(v), is_short);
#pragma unroll
                for (int i = 0; i < kLot; i++) n[v].x[i] = !TAIL || i < left ? (n[v].x[i] - mean_a) * rstd_a : 0.f;
                if (p.before.kind == FTC_NORM_NONE) continue;
                if (p.residual.ptr) xh[v] = widen<TAIL, MOVE>(residual_raw[v], type_of<DS>(p.residual), p.D - column(v), is_short);
                if (p.grad_h.ptr) dx[v] = widen<TAIL, MOVE>(gh_raw[v], type_of<DB>(p.grad_h), p.D - column(v), is_short);
                Lot w, b;
                params_lot<TAIL, MOVE>(p.after, col, left, is_short, w, b);
#pragma unroll
                for (int i = 0; i < kLot; i++) {
                    const float y = fmaf(n[v].x[i], w.x[i], b.x[i]);
                    float value = 1.f, slope;
                    if (p.gate.ptr) activate(gate[v].x[i], p.activation, value, slope);
                    const float a = value * y;
                    xh[v].x[i] = !TAIL || i < left ? (fmaf(p.scale, a, xh[v].x[i]) - mean_b) * rstd_b : 0.f;
                }
                params_lot<TAIL, MOVE>(p.before, col, left, is_short, w, b);
#pragma unroll
                for (int i = 0; i < kLot; i++) {
                    dwb[v].x[i] = fmaf(dx[v].x[i], xh[v].x[i], dwb[v].x[i]);
                    if (FULL) dbb[FULL ? v : 0].x[i] += dx[v].x[i];
                    dx[v].x[i] *= w.x[i];
                    s0 += dx[v].x[i];
                    s1 = fmaf(dx[v].x[i], xh[v].x[i], s1);
                }
            }
            if (p.before.kind != FTC_NORM_NONE) {
                team_sum<LPR>(s0, s1, mem, turn);
                s0 = p.before.kind == FTC_NORM_LAYER ? s0 * per : 0.f, s1 *= per;
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int i = 0; i < kLot; i++) dx[v].x[i] = rstd_b * ((dx[v].x[i] - s0) - xh[v].x[i] * s1);
            }
            float t0 = 0.f, t1 = 0.f;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int col = column(v), left = p.D - col;
                if (!live || col >= p.D) continue;
                if (p.grad_x.ptr) {
                    const Lot g = widen<TAIL, MOVE>(gx_raw[v], type_of<DS>(p.grad_x), p.D - column(v), is_short);
#pragma unroll
                    for (int i = 0; i < kLot; i++) dx[v].x[i] += g.x[i];
                }
                if (TAIL)
#pragma unroll
                    for (int i = 0; i < kLot; i++) dx[v].x[i] = i < left ? dx[v].x[i] : 0.f;
                if (p.grad_residual.ptr)
                    store_lot<TAIL>(p.grad_residual.ptr, type_of<DS>(p.grad_residual), row * p.grad_residual.stride + col, left, dx[v]);
                Lot w, b;
                params_lot<TAIL, MOVE>(p.after, col, left, is_short, w, b);
                if (p.gate.ptr) {
                    Lot d;
#pragma unroll
                    for (int i = 0; i < kLot; i++) {
                        const float y = fmaf(n[v].x[i], w.x[i], b.x[i]);
                        float value, slope;
                        activate(gate[v].x[i], p.activation, value, slope);
                        d.x[i] = p.scale * slope * y * dx[v].x[i];
                        dx[v].x[i] *= p.scale * value;
                        if (FULL) dgate[FULL ? v : 0].x[i] += d.x[i];
                    }
                    if (p.grad_gate.ptr && !(FULL && p.shared))
                        store_lot<TAIL>(p.grad_gate.ptr, type_of<DB>(p.grad_gate), row * p.grad_gate.stride + col, left, d);
                } else {
#pragma unroll
                    for (int i = 0; i < kLot; i++) dx[v].x[i] *= p.scale;
                }
                if (p.after.kind == FTC_NORM_NONE) continue;
#pragma unroll
                for (int i = 0; i < kLot; i++) {
                    dwa[v].x[i] = fmaf(dx[v].x[i], n[v].x[i], dwa[v].x[i]);
                    if (FULL) dba[FULL ? v : 0].x[i] += dx[v].x[i];
                    dx[v].x[i] *= w.x[i];
                    t0 += dx[v].x[i];
                    t1 = fmaf(dx[v].x[i], n[v].x[i], t1);
                }
            }
            if (p.after.kind != FTC_NORM_NONE) {
                team_sum<LPR>(t0, t1, mem, turn);
                t0 = p.after.kind == FTC_NORM_LAYER ? t0 * per : 0.f, t1 *= per;
#pragma unroll
                for (int v = 0; v < NV; v++)
#pragma unroll
                    for (int i = 0; i < kLot; i++) dx[v].x[i] = rstd_a * ((dx[v].x[i] - t0) - n[v].x[i] * t1);
            }
            if (p.grad_block.ptr && live)
#pragma unroll
                for (int v = 0; v < NV; v++)
                    if (column(v) < p.D)
                        store_lot<TAIL>(p.grad_block.ptr, type_of<DB>(p.grad_block), row * p.grad_block.stride + column(v),
                                       p.D - column(v), dx[v]);
        }
        if constexpr (FULL)
            if (p.gate_sums) leave(dgate, p.gate_sums + (seg * p.parts + part) * p.D);
    }
    float *const to = p.sums + (int64_t)blockIdx.x * kSums * p.D;
    if (p.sums && p.after.weight) leave(dwa, to + kAfterWeight * p.D);
    if constexpr (FULL)
        if (p.sums && p.after.bias) leave(dba, to + kAfterBias * p.D);
    if (p.sums && p.before.weight) leave(dwb, to + kBeforeWeight * p.D);
    if constexpr (FULL)
        if (p.sums && p.before.bias) leave(dbb, to + kBeforeBias * p.D);
}

// ---- launches ----
// Whether the backward needs the kernel that sums biases and shared gates as well
inline bool full(const Args &p) { return p.after.bias || p.before.bias || p.shared; }

struct Plan {
    int lpr, teams;
    int64_t groups, parts;  // workgroups, workgroups per segment
};

// BACKWARD, TAIL: one translation unit instantiates the kernels of each
template <int LPR, int NV, bool BACKWARD, bool TAIL, int DB, int DS>
void launch(const Args &p, const Plan &q, hipStream_t stream) {
    const dim3 grid((uint32_t)q.groups), block(LPR > 256 ? LPR : 256);
    if constexpr (!BACKWARD) residual_norm_kernel<LPR, NV, TAIL, DB, DS><<<grid, block, 0, stream>>>(p);
    else if (full(p)) residual_norm_backward_kernel<LPR, NV, TAIL, DB, DS, true><<<grid, block, 0, stream>>>(p);
    else residual_norm_backward_kernel<LPR, NV, TAIL, DB, DS, false><<<grid, block, 0, stream>>>(p);
}
template <int LPR, int NV, bool BACKWARD, bool TAIL>
void launch(const Args &p, const Plan &q, hipStream_t stream) {
    // the type that all the rows of a side have, or -1
    auto common = [](std::initializer_list<const Rows *> rows, int otherwise) {
        int type = otherwise;
        for (const Rows *r : rows)
            if (r->ptr) type = type == otherwise || type == r->dtype ? r->dtype : -2;
        return type;
    };
    const int b = common({&p.block, &p.gate, &p.h, &p.grad_h, &p.grad_block, &p.grad_gate}, -1);
    const int s = common({&p.residual, &p.x, &p.grad_x, &p.grad_residual}, -1);
    const int stream_type = s == -1 ? b : s;  // (no rows of that side at all: any will do)
    if (b == FTC_F32 && stream_type == FTC_F32) launch<LPR, NV, BACKWARD, TAIL, FTC_F32, FTC_F32>(p, q, stream);
    else if (b == FTC_BF16 && stream_type == FTC_BF16) launch<LPR, NV, BACKWARD, TAIL, FTC_BF16, FTC_BF16>(p, q, stream);
    else if (b == FTC_BF16 && stream_type == FTC_F32) launch<LPR, NV, BACKWARD, TAIL, FTC_BF16, FTC_F32>(p, q, stream);
    else launch<LPR, NV, BACKWARD, TAIL, -1, -1>(p, q, stream);
}
template <bool BACKWARD, bool TAIL>
void dispatch(const Args &p, const Plan &q, hipStream_t stream) {
    if (p.D <= 128) launch<16, 1, BACKWARD, TAIL>(p, q, stream);
    else if (p.D <= 512) launch<64, 1, BACKWARD, TAIL>(p, q, stream);
    else if (p.D <= 1024) launch<128, 1, BACKWARD, TAIL>(p, q, stream);
    else if (p.D <= 2048) launch<256, 1, BACKWARD, TAIL>(p, q, stream);
    else if (p.D <= 4096) launch<512, 1, BACKWARD, TAIL>(p, q, stream);
    else if (p.D <= 8192) launch<512, 2, BACKWARD, TAIL>(p, q, stream);
    else launch<1024, 2, BACKWARD, TAIL>(p, q, stream);
}

// (TAIL: rows whose width is not a multiple of kLot)
void norm_forward(const Args &p, const Plan &q, hipStream_t stream);
void norm_forward_tail(const Args &p, const Plan &q, hipStream_t stream);
void norm_backward(const Args &p, const Plan &q, hipStream_t stream);
void norm_backward_tail(const Args &p, const Plan &q, hipStream_t stream);

}  // namespace norm
}  // namespace ftc
