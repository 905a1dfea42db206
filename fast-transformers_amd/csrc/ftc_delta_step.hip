// The gated delta rule position by position, on the vector unit: the step of decoding, and calls of a few positions.
//
//   S' = e^g S,  (a, b) = (S'^T k^, S'^T q^),  u = beta (v - a),  o = b + (k^ . q^) u,  S <- S' + k^ u^T
//
// (o = S^T q^ of the new state: both products read the faded one, so a position is one pass and one reduction.)
//
// What bounds it is the state, read and written once per call (8 E M bytes a chain), and on few chains latency.  A
// workgroup of 256 lanes owns 64 columns of one chain's state in registers: 64 / VEC lanes side by side (VEC = 4:
// 16-byte accesses), the others take every kGroups-th row.  Sums are in a fixed order, everything is fp32.
// Measured: 4096 chains of 128 x 128 107 us, 5.0 TB/s of states; 8 chains of 64 x 64 6 us, of which a launch is 4.
#include "ftc_delta_kernel.h"

namespace ftc {
namespace delta {
namespace {

constexpr int kLanes = 256, kBlock = 64;

template <int VEC>
struct Cells {
    float x[VEC];
};

// RPL: rows of the state per lane
template <int VEC, int RPL>
__global__ __launch_bounds__(kLanes) void delta_step_kernel(DeltaArgs p) {
    constexpr int kAcross = kBlock / VEC, kGroups = kLanes / kAcross, kWaves = kLanes / 64;
    __shared__ float k_mem[kMaxE], q_mem[kMaxE];
    __shared__ float part_mem[2][kWaves][kBlock];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int across = tid % kAcross, group = tid / kAcross;
    const int blocks = (p.M + kBlock - 1) / kBlock;
    const Where w = where_of(p, (int)(blockIdx.x / (uint32_t)blocks), 0);
    const int col = (int)(blockIdx.x % (uint32_t)blocks) * kBlock + across * VEC;
    const bool mine = col < p.M;  // (VEC = 4: M is a multiple of 4)

    Cells<VEC> S[RPL];
#pragma unroll
    for (int i = 0; i < RPL; i++) {
        const int e = group + kGroups * i;
#pragma unroll
        for (int j = 0; j < VEC; j++) S[i].x[j] = 0.f;
        if (p.initial.ptr && mine && e < p.E) {
            const float *const from = p.initial.ptr + w.n * p.initial.stride_n + w.h * p.initial.stride_h + e * p.initial.stride_d + col;
            if (VEC == 4) {
                const f32x4 t = *(const f32x4a *)from;
#pragma unroll
                for (int j = 0; j < VEC; j++) S[i].x[j] = t[j % 4];
            } else {
                S[i].x[0] = from[0];
            }
        }
    }
    auto row_at = [&](const Operand &o, int h, int l) { return w.n * o.stride_n + h * o.stride_h + (int64_t)l * o.stride_l; };
    for (int l = 0; l < w.len; l++) {
        // the rows of k and q in LDS, and their three products, by every wavefront for itself
        float k0 = 0.f, k1 = 0.f, q0 = 0.f, q1 = 0.f;
        if (lane < p.E) {
            k0 = load_as_f32(p.k.ptr, p.k.dtype, row_at(p.k, w.hk, l) + lane);
            q0 = load_as_f32(p.q.ptr, p.q.dtype, row_at(p.q, w.hk, l) + lane);
        }
        if (lane + 64 < p.E) {
            k1 = load_as_f32(p.k.ptr, p.k.dtype, row_at(p.k, w.hk, l) + lane + 64);
            q1 = load_as_f32(p.q.ptr, p.q.dtype, row_at(p.q, w.hk, l) + lane + 64);
        }
        const float g = load_as_f32(p.g.ptr, p.g.dtype, w.n * p.g.sn + w.h * p.g.sh + l * p.g.sl);
        const float beta = load_as_f32(p.b.ptr, p.b.dtype, w.n * p.b.sn + w.h * p.b.sh + l * p.b.sl);
        float v[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++)
            v[j] = mine ? load_as_f32(p.v.ptr, p.v.dtype, row_at(p.v, w.h, l) + col + j) : 0.f;
        float kk = fmaf(k0, k0, k1 * k1), qq = fmaf(q0, q0, q1 * q1), kq = fmaf(k0, q0, k1 * q1);
#pragma unroll
        for (int d = 1; d < 64; d *= 2) kk += __shfl_xor(kk, d), qq += __shfl_xor(qq, d), kq += __shfl_xor(kq, d);
        const float rk = p.normalize ? 1.f / sqrtf(kk + kNormEps) : 1.f;
        const float rq = p.normalize ? p.scale / sqrtf(qq + kNormEps) : p.scale;
        if (wave == 0) {
            k_mem[lane] = k0 * rk, q_mem[lane] = q0 * rq;
            k_mem[lane + 64] = k1 * rk, q_mem[lane + 64] = q1 * rq;
        }
        __syncthreads();
        const float fade = expf(g);
        float a[VEC], b[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) a[j] = b[j] = 0.f;
#pragma unroll
        for (int i = 0; i < RPL; i++) {
            const float ke = k_mem[group + kGroups * i], qe = q_mem[group + kGroups * i];
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                S[i].x[j] *= fade;
                a[j] = fmaf(ke, S[i].x[j], a[j]);
                b[j] = fmaf(qe, S[i].x[j], b[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) {
#pragma unroll
            for (int d = kAcross; d < 64; d *= 2) a[j] += __shfl_xor(a[j], d), b[j] += __shfl_xor(b[j], d);
            if (lane < kAcross) part_mem[0][wave][across * VEC + j] = a[j], part_mem[1][wave][across * VEC + j] = b[j];
        }
        __syncthreads();
        float u[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const int x = across * VEC + j;
            a[j] = (part_mem[0][0][x] + part_mem[0][1][x]) + (part_mem[0][2][x] + part_mem[0][3][x]);
            u[j] = beta * (v[j] - a[j]);
        }
        if (mine && tid < kAcross) {
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const int x = across * VEC + j;
                const float bj = (part_mem[1][0][x] + part_mem[1][1][x]) + (part_mem[1][2][x] + part_mem[1][3][x]);
                store_from_f32(p.out.ptr, p.out.dtype,
                               w.n * p.out.stride_n + w.h * p.out.stride_h + (int64_t)l * p.out.stride_l + col + j,
                               fmaf(kq * rk * rq, u[j], bj));
            }
        }
#pragma unroll
        for (int i = 0; i < RPL; i++) {
            const float ke = k_mem[group + kGroups * i];
#pragma unroll
            for (int j = 0; j < VEC; j++) S[i].x[j] = fmaf(ke, u[j], S[i].x[j]);
        }
        __syncthreads();  // (k_mem and part_mem are written again)
    }
    if (mine && tid < kAcross)
        for (int l = w.len; l < p.L; l++)
#pragma unroll
            for (int j = 0; j < VEC; j++)
                store_from_f32(p.out.ptr, p.out.dtype,
                               w.n * p.out.stride_n + w.h * p.out.stride_h + (int64_t)l * p.out.stride_l + col + j, 0.f);
    if (!p.final_.ptr || !mine) return;
#pragma unroll
    for (int i = 0; i < RPL; i++) {
        const int e = group + kGroups * i;
        if (e >= p.E) continue;
        float *const to = p.final_.ptr + w.n * p.final_.stride_n + w.h * p.final_.stride_h + e * p.final_.stride_d + col;
        if (VEC == 4) *(f32x4a *)to = f32x4{S[i].x[0], S[i].x[1 % VEC], S[i].x[2 % VEC], S[i].x[3 % VEC]};
        else to[0] = S[i].x[0];
    }
}

bool state_vec(const StateRef &s) {
    return !s.ptr || (((uintptr_t)s.ptr & 15) == 0 && s.stride_n % 4 == 0 && s.stride_h % 4 == 0 && s.stride_d % 4 == 0);
}

}  // namespace

int delta_steps(const DeltaArgs &p, hipStream_t stream) {
    const dim3 grid((uint32_t)p.N * (uint32_t)p.H * (uint32_t)((p.M + kBlock - 1) / kBlock));
    const bool vec = p.M % 4 == 0 && state_vec(p.initial) && state_vec(p.final_);
    if (vec) {
        if (p.E <= 64) delta_step_kernel<4, 4><<<grid, kLanes, 0, stream>>>(p);
        else delta_step_kernel<4, 8><<<grid, kLanes, 0, stream>>>(p);
    } else {
        if (p.E <= 64) delta_step_kernel<1, 16><<<grid, kLanes, 0, stream>>>(p);
        else delta_step_kernel<1, 32><<<grid, kLanes, 0, stream>>>(p);
    }
    return FTC_OK;
}

}  // namespace delta
}  // namespace ftc
