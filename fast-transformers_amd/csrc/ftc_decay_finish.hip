// Decayed linear attention, behind the scans: the states at the segments' borders from what each segment writes, the gradients of
// the log decays from what every position receives and sends, and the gradients of shared queries and keys from their shares.
// Formulas: ftc_decay_kernel.h.  All sums are in a fixed order.  What bounds them is latency: borders 8.3 us for 128 chains of four segments
// of 128 x 128 (50 MB, 6.1 TB/s, some of it from the last cache), 10.2 for 16 of 43 of 64 x 64 (six reads of eight, one after the other); the gradients of log decays 15 us for 128 chains
// of 4096 positions (9.5 MB; sums in 64 bits), 6.4 for 80 of 1000, and 4.6 more where they are those of heads.
#include "ftc_decay_kernel.h"

namespace ftc {
namespace decay {
namespace {

constexpr int kThreads = 256;
constexpr int kMostChunks = kLongest / kRows;
// log decay of a chunk behind which nothing of what came before is left: e^-21 is 2^-30
constexpr double kShut = -21.0;

// slot <- slot + e^{total} (slot before it), from border to border; those of the next eight are on their way meanwhile
__global__ __launch_bounds__(kThreads) void decay_borders_kernel(float *slots, const double *totals, int64_t chains, int segments, int slices,
                                                                 int size, int reverse) {
    constexpr int kAhead = 8;
    const int per = (size / 4 + kThreads - 1) / kThreads;
    const int64_t chain = blockIdx.x / per;
    const int i = 4 * ((int)(blockIdx.x - chain * per) * kThreads + threadIdx.x);
    if (i >= size) return;
    float *const at = slots + chain * (segments + 1) * size + i;
    const double *const sums = totals + chain / slices * segments;
    // the n-th on the way: its border, and the segment in front of it
    auto border = [&](int n) { return at + (int64_t)(reverse ? segments - 1 - n : n + 1) * size; };
    auto factor = [&](int n) {
        const double x = sums[reverse ? segments - 1 - n : n] * 1.4426950408889634;
        return power((float)x, (float)(x - (double)(float)x));
    };
    f32x4 x = *(const f32x4a *)border(0);
    for (int n0 = 1; n0 < segments - 1; n0 += kAhead) {
        f32x4 own[kAhead];
        float by[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const int n = min(n0 + k, segments - 2);
            own[k] = *(const f32x4a *)border(n), by[k] = factor(n);
        }
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            if (n0 + k < segments - 1) {
#pragma unroll
                for (int r = 0; r < 4; r++) x[r] = fmaf(by[k], x[r], own[k][r]);
                *(f32x4a *)border(n0 + k) = x;
            }
    }
}

// X of a segment's positions.  A workgroup takes one segment of one head, the chains of its slices together, a wavefront a
// chunk of it.
__global__ __launch_bounds__(64 * kMostChunks) void decay_finish_kernel(FinishArgs p) {
    __shared__ double gets_mem[kMostChunks], sends_mem[kMostChunks], through_mem[kMostChunks], more_mem[kMostChunks];
    __shared__ bool shut_mem[kMostChunks];
    const int lane = threadIdx.x & 63, wave = scalar(threadIdx.x >> 6);
    const int head = (int)(blockIdx.x / p.segments), seg = (int)(blockIdx.x - head * p.segments);
    const int n = head / p.H, h = head - n * p.H;
    int64_t len = p.lengths ? p.lengths[n] : p.L;
    len = len < 0 ? 0 : len > p.L ? p.L : len;
    const int64_t start = (int64_t)seg * p.seg_len, stop = min(start + p.seg_len, (int64_t)p.L), end = min(stop, len);
    const int chunks = end > start ? (int)((end - start + kRows - 1) / kRows) : 0;
    const int64_t chains = (int64_t)p.N * p.H * p.slices, chain = (int64_t)head * p.slices;
    auto sum64 = [](double x) {
#pragma unroll
        for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
        return x;
    };
    const int64_t l = start + kRows * wave + lane;
    const bool live = l < end;
    // what position l receives and sends, from and to other chunks, and altogether
    double gets = 0.0, sends = 0.0, gets_all = 0.0, sends_all = 0.0;
    float decay = 0.f;
    if (live) {
        const int64_t step = chains * p.L;
        for (int s = 0; s < p.slices; s++) {
            const int64_t at = (chain + s) * p.L + l;
            gets += (double)p.x[at], gets_all += (double)p.x[at + step];
            sends += (double)p.y[at], sends_all += (double)p.y[at + step];
        }
        decay = load_as_f32(p.g.ptr, p.g.dtype, n * p.g.sn + h * p.g.sh + l * p.g.sl);
    }
    if (wave < chunks) {
        const double all_gets = sum64(gets), all_sends = sum64(sends), all = sum64(live ? fmax((double)decay, -1000.0) : 0.0);
        if (lane == 0) gets_mem[wave] = all_gets, sends_mem[wave] = all_sends, shut_mem[wave] = all < kShut;
    }
    __syncthreads();
    if (wave == 0 && chunks > 0) {
        // X at the segment's borders, a share a lane
        double at_border[2];
#pragma unroll
        for (int b = 0; b < 2; b++) {
            double x = 0.0;
            for (int i = lane; i < p.slices * p.shares; i += 64)
                x += p.anchors[((chain + i / p.shares) * (p.segments + 1) + seg + b) * p.shares + i % p.shares];
            at_border[b] = sum64(x);
        }
        if (lane == 0) {
            // What crosses a whole chunk: X at its first position but for what the chunk receives; with what it sends that is X at
            // the next one's.  The roundings of those sums add up until X is known again, before a chunk that nothing crosses
            // or at the segment's end, and what they come to then is spread over the positions since.
            double x = at_border[0];
            int known = 0;
            for (int k = 0; k <= chunks; k++) {
                const bool ends = k == chunks;
                if (!ends && !shut_mem[k]) {
                    through_mem[k] = x - gets_mem[k], more_mem[k] = 0.0, x = through_mem[k] + sends_mem[k];
                    continue;
                }
                const double each = k > known ? (x - (ends ? at_border[1] : gets_mem[k])) / (k - known) : 0.0;
                for (int i = known; i < k; i++) through_mem[i] -= each * (i - known), more_mem[i] = each;
                if (!ends) through_mem[k] = more_mem[k] = 0.0, x = sends_mem[k];
                known = k + 1;
            }
        }
    }
    __syncthreads();
    double x = 0.0;
    if (wave < chunks) {
        // (within the chunk all that is sent is received: what the sums differ by is rounding)
        const double count = (double)min((int64_t)kRows, end - start - kRows * wave);
        double within = (sends_all - sends) - (gets_all - gets);
        const double differ = sum64(within);
        within -= live ? differ / count : 0.0;
        const double own = within + sends - gets;
        x = own;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double other = __shfl_up(x, d);
            if (lane >= d) x += other;
        }
        x += (through_mem[wave] + gets_mem[wave]) - own - more_mem[wave] * (lane / count);
        if (!live || decay == -INFINITY) x = 0.0;  // (behind a decay of -infinity nothing depends on it)
    }
    if (!p.per_head) {
        if (l < stop) store_from_f32(p.gg.ptr, p.gg.dtype, n * p.gg.sn + h * p.gg.sh + l * p.gg.sl, (float)x);
        return;
    }
    x = sum64(x);
    __syncthreads();
    if (lane == 0) gets_mem[wave] = x;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = 0.0;
        for (int k = 0; k < chunks; k++) total += gets_mem[k];
        p.sums[(int64_t)h * p.N * p.segments + (int64_t)n * p.segments + seg] = total;
    }
}
__global__ __launch_bounds__(64) void decay_heads_kernel(FinishArgs p) {
    const int count = p.N * p.segments;
    const double *const from = p.sums + (int64_t)blockIdx.x * count;
    double x = 0.0;
    for (int i = threadIdx.x; i < count; i += 64) x += from[i];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
    if (threadIdx.x == 0) store_from_f32(p.gg.ptr, p.gg.dtype, blockIdx.x * p.gg.sh, (float)x);
}

// The gradients of rows that several chains read, where no two of them share a workgroup (ftc_decay.hip), bound by memory.  LOT: values that a
// lane takes at a time, four where the rows' widths and places allow it.  (4 sequences of 2048, 16 heads on 4 key heads of 64, fp32, with
// all of the backward: 228 us, by single values 250.)
template <int LOT>
__global__ __launch_bounds__(kThreads) void decay_gather_kernel(FinishArgs p) {
    const int which = blockIdx.y;
    const float *const part = p.part[which];
    const OperandOut &to = p.sum[which];
    if (!part) return;
    const int group = p.H * p.slices / p.Hk / p.every;
    const int64_t size = (int64_t)p.L * p.E;
    const int64_t per = (size / LOT + kThreads - 1) / kThreads;
    for (int64_t block = blockIdx.x; block < (int64_t)p.N * p.Hk * per; block += gridDim.x) {
        const int64_t chain = block / per, rest = LOT * ((block - chain * per) * kThreads + threadIdx.x);
        if (rest >= size) continue;
        const int64_t l = size < (1ll << 31) ? (int64_t)((uint32_t)rest / (uint32_t)p.E) : rest / p.E, e = rest - l * p.E;
        const float *const from = part + chain * group * size + rest;
        float x[LOT];
#pragma unroll
        for (int i = 0; i < LOT; i++) x[i] = 0.f;
        for (int g = 0; g < group; g++) {
            if constexpr (LOT == 4) {
                const f32x4 y = *(const f32x4a *)(from + g * size);
#pragma unroll
                for (int i = 0; i < LOT; i++) x[i] += y[i];
            } else {
                x[0] += from[g * size];
            }
        }
        const int64_t n = chain / p.Hk, h = chain - n * p.Hk, at = n * to.stride_n + h * to.stride_h + l * to.stride_l + e;
        if constexpr (LOT == 4) {
            if (to.dtype == FTC_F32) *(f32x4a *)((float *)to.ptr + at) = f32x4{x[0], x[1], x[2], x[3]};
            else *(u32x2a *)((uint16_t *)to.ptr + at) = u32x2{delta::to_bf16(x[0], x[1]), delta::to_bf16(x[2], x[3])};
        } else {
            store_from_f32(to.ptr, to.dtype, at, x[0]);
        }
    }
}

}  // namespace

void decay_borders(const Args &p, const Task &task, hipStream_t stream) {
    const int size = p.slot_rows * p.width;
    const int64_t chains = (int64_t)p.N * p.H * p.slices;
    decay_borders_kernel<<<dim3((uint32_t)(chains * ((size / 4 + kThreads - 1) / kThreads))), kThreads, 0, stream>>>(
        task.slots, p.totals, chains, p.segments, p.slices, size, task.reverse);
}
void decay_finish(const FinishArgs &p, hipStream_t stream) {
    decay_finish_kernel<<<dim3((uint32_t)(p.N * p.H * p.segments)), p.seg_len, 0, stream>>>(p);
    if (p.per_head) decay_heads_kernel<<<dim3((uint32_t)p.H), 64, 0, stream>>>(p);
}
void decay_gather(const FinishArgs &p, hipStream_t stream) {
    bool four = p.E % 4 == 0;
    for (const OperandOut &o : p.sum) {
        const int lot = o.dtype == FTC_F32 ? 16 : 8;
        four = four && (!o.ptr || (o.stride_n % 4 == 0 && o.stride_h % 4 == 0 && o.stride_l % 4 == 0 && (uintptr_t)o.ptr % lot == 0));
    }
    const int64_t size = (int64_t)p.L * p.E / (four ? 4 : 1);
    const int64_t blocks = (int64_t)p.N * p.Hk * ((size + kThreads - 1) / kThreads);
    const dim3 grid((uint32_t)(blocks < (1 << 22) ? blocks : 1 << 22), 2);
    if (four) decay_gather_kernel<4><<<grid, kThreads, 0, stream>>>(p);
    else decay_gather_kernel<1><<<grid, kThreads, 0, stream>>>(p);
}

}  // namespace decay
}  // namespace ftc
