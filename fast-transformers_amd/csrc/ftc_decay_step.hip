// Decayed linear attention position by position, on the vector unit: the step of decoding, and calls of a few positions.
//
//   S <- e^g S + k v^T,   o = scale S^T q
//
// What bounds it is the state, read and written once per call (8 E M bytes a chain), and on few chains latency.  A
// workgroup owns 64 columns of one chain's state in registers: 64 / VEC lanes side by side (VEC = 4: 16-byte accesses), and
// sixteen such groups that take every sixteenth row.  Sums are in a fixed order, everything is fp32.
//
// 4096 chains of 128 x 128: 89 us in a graph, 540 MB, 6.0 TB/s (half of the states stay in the last cache from one step to the next),
// 105 on states that are not there; by single values, for states that lie otherwise, 149.  8 chains of 64 x 64: 4.5 and 4.9.
#include "ftc_decay_kernel.h"

namespace ftc {
namespace decay {
namespace {

constexpr int kBlock = 64, kGroups = 16;

// RPL: rows of the state per lane
template <int VEC, int RPL>
__global__ __launch_bounds__(kGroups * kBlock / VEC) void decay_step_kernel(StepArgs p) {
    constexpr int kAcross = kBlock / VEC, kWaves = kGroups * kAcross / 64;
    __shared__ float part_mem[kWaves][kBlock], k_mem[kMaxE], q_mem[kMaxE];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int across = tid % kAcross, group = tid / kAcross;
    const int blocks = (p.M + kBlock - 1) / kBlock;
    const int chain = scalar((int)(blockIdx.x / (uint32_t)blocks)), n = scalar(chain / p.H), h = chain - n * p.H;
    const int hk = scalar(h / (p.H / p.Hk));
    int64_t length = p.lengths ? p.lengths[n] : p.L;
    const int len = (int)(length < 0 ? 0 : length > p.L ? p.L : length);
    const int col = (int)(blockIdx.x % (uint32_t)blocks) * kBlock + across * VEC;
    const bool mine = col < p.M;  // (VEC = 4: M is a multiple of 4)

    float S[RPL][VEC];
#pragma unroll
    for (int i = 0; i < RPL; i++) {
        const int e = group + kGroups * i;
#pragma unroll
        for (int j = 0; j < VEC; j++) S[i][j] = 0.f;
        if (p.first.ptr && mine && e < p.E) {
            const float *const from = p.first.ptr + n * p.first.sn + h * p.first.sh + e * p.first.sd + col;
            if (VEC == 4) {
                const f32x4 t = *(const f32x4a *)from;
#pragma unroll
                for (int j = 0; j < VEC; j++) S[i][j] = t[j % 4];
            } else {
                S[i][0] = from[0];
            }
        }
    }
    auto row_at = [&](const Operand &o, int head, int l) { return n * o.stride_n + head * o.stride_h + (int64_t)l * o.stride_l; };
    for (int l = 0; l < len; l++) {
        const float g = load_as_f32(p.g.ptr, p.g.dtype, n * p.g.sn + h * p.g.sh + l * p.g.sl);
        float v[VEC], o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) v[j] = mine ? load_as_f32(p.v.ptr, p.v.dtype, row_at(p.v, h, l) + col + j) : 0.f, o[j] = 0.f;
        if (tid < 2 * kMaxE) {
            const int e = tid & (kMaxE - 1);
            const Operand &row = tid < kMaxE ? p.k : p.q;
            (tid < kMaxE ? k_mem : q_mem)[e] = e < p.E ? load_as_f32(row.ptr, row.dtype, row_at(row, hk, l) + e) : 0.f;
        }
        __syncthreads();
        const float fade = expf(g);
#pragma unroll
        for (int i = 0; i < RPL; i++) {
            const float k = k_mem[group + kGroups * i], q = q_mem[group + kGroups * i];
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                S[i][j] = fmaf(k, v[j], fade * S[i][j]);
                o[j] = fmaf(q, S[i][j], o[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) {
#pragma unroll
            for (int d = kAcross; d < 64; d *= 2) o[j] += __shfl_xor(o[j], d);
            if (lane < kAcross) part_mem[wave][across * VEC + j] = o[j];
        }
        __syncthreads();
        if (mine && tid < kAcross) {
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const int x = across * VEC + j;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < kWaves; i++) sum += part_mem[i][x];
                store_from_f32(p.out.ptr, p.out.dtype, n * p.out.stride_n + h * p.out.stride_h + (int64_t)l * p.out.stride_l + col + j,
                               p.scale * sum);
            }
        }
        __syncthreads();  // (the rows and part_mem are written again)
    }
    if (mine && tid < kAcross)
        for (int l = len; l < p.L; l++)
#pragma unroll
            for (int j = 0; j < VEC; j++)
                store_from_f32(p.out.ptr, p.out.dtype,
                               n * p.out.stride_n + h * p.out.stride_h + (int64_t)l * p.out.stride_l + col + j, 0.f);
    if (!p.last.ptr || !mine) return;
#pragma unroll
    for (int i = 0; i < RPL; i++) {
        const int e = group + kGroups * i;
        if (e >= p.E) continue;
        float *const to = p.last.ptr + n * p.last.sn + h * p.last.sh + e * p.last.sd + col;
        if (VEC == 4) *(f32x4a *)to = f32x4{S[i][0], S[i][1 % VEC], S[i][2 % VEC], S[i][3 % VEC]};
        else to[0] = S[i][0];
    }
}

bool state_vec(const State &s) {
    return !s.ptr || (((uintptr_t)s.ptr & 15) == 0 && s.sn % 4 == 0 && s.sh % 4 == 0 && s.sd % 4 == 0);
}

}  // namespace

bool decay_step_vec(const StepArgs &p) { return p.M % 4 == 0 && state_vec(p.first) && state_vec(p.last); }
int64_t decay_step_lanes(int64_t chains, int64_t M, bool vec) { return chains * ((M + kBlock - 1) / kBlock) * (kGroups * kBlock / (vec ? 4 : 1)); }
void decay_steps(const StepArgs &p, hipStream_t stream) {
    const dim3 grid((uint32_t)p.N * (uint32_t)p.H * (uint32_t)((p.M + kBlock - 1) / kBlock));
    if (decay_step_vec(p)) {
        if (p.E <= 64) decay_step_kernel<4, 4><<<grid, 256, 0, stream>>>(p);
        else decay_step_kernel<4, 8><<<grid, 256, 0, stream>>>(p);
    } else {
        if (p.E <= 64) decay_step_kernel<1, 4><<<grid, 1024, 0, stream>>>(p);
        else decay_step_kernel<1, 8><<<grid, 1024, 0, stream>>>(p);
    }
}

}  // namespace decay
}  // namespace ftc
