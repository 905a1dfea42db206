// The gated delta rule, what the chunks need of the keys, decays and beta alone: the row factors and
// T = (I + M)^-1 of every chunk (formulas and layouts: ftc_delta_kernel.h).
//
// One workgroup of four wavefronts per chunk and chain.  The inverse of the unit lower triangular matrix of 64 rows
// is made from its four diagonal blocks of 16 by substitution (a lane per column, in registers), then of 32 and 64
// from T21 = -T22 (M21 T11) on the fp32 matrix instruction.  (Products of powers of M would be fewer steps, but for
// keys that resemble each other their entries grow to binomials that cancel.)
//
// What bounds it: the steps of the inverse one after the other, and what it writes (36 KB of T and its transpose a chunk, 32 KB of
// the keys' fragments).  T lies where k was, so that three workgroups fit a compute unit.  Measured: 8192 chunks
// of 128 key columns, bf16, 181 us (2.5 TB/s written; two workgroups a compute unit 220; 250
// to 300 where a backward follows and every chunk has betas of zero, since T is then made twice); 1280 of 64, fp32, 38.
#include "ftc_delta_kernel.h"

namespace ftc {
namespace delta {
namespace {

constexpr int kThreads = 256;
constexpr int kStride = 68;  // floats per row of the square matrices in LDS: rows 4 banks apart

__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// sum of squares of 64 rows, one value per row of the tile, to `to`
template <typename T, int COLS>
__device__ __forceinline__ void squares(const RowTile<T, COLS, kThreads> &tile, lds_float *to, int tid) {
    using Tile = RowTile<T, COLS, kThreads>;
#pragma unroll
    for (int i = 0; i < Tile::kPer; i++) {
        float s = 0.f;
#pragma unroll
        for (int x = 0; x < 8; x++) s = fmaf(tile.value(i, x), tile.value(i, x), s);
#pragma unroll
        for (int d = 1; d < Tile::kAcross; d *= 2) s += __shfl_xor(s, d);
        const int u = tid + kThreads * i;
        if (u % Tile::kAcross == 0) to[u / Tile::kAcross] = s;
    }
}

template <typename T, int KE>
__global__ __launch_bounds__(kThreads) void delta_prepare_kernel(DeltaArgs p) {
    constexpr int RB = 64 * KE, PIECES = Elem<T>::kPieces;
    using Tile = RowTile<T, 32 * KE, kThreads>;
    // k, and T where it was; M and what is made of it, and at the end T's three planes there
    constexpr int kPlanes = PIECES * Plane<RB>::kBytes, kT = 4 * kRows * kStride, kM = kT + 4 * 32 * kStride;
    __shared__ __align__(16) char k_mem[kPlanes > kT ? kPlanes : kT], m_mem[kM > 3 * Plane<128>::kBytes ? kM : 3 * Plane<128>::kBytes];
    __shared__ float k2_mem[kRows], q2_mem[kRows], high_mem[kRows], low_mem[kRows], beta_mem[2][kRows], rk_mem[kRows];
    __shared__ int again_mem;
    lds_char *const kp = (lds_char *)k_mem;
    lds_float *const Mx = (lds_float *)m_mem, *const Tm = (lds_float *)k_mem, *const X = Mx + kRows * kStride;

    int tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4;
    const int wave = scalar(tid >> 6);
    const Where w = where_of(p, (int)(blockIdx.x / (uint32_t)p.chunks), (int)(blockIdx.x % (uint32_t)p.chunks));
    if (w.valid == 0) return;  // (nobody reads what belongs to it)
    const int64_t l0 = (int64_t)w.chunk * kRows;

    Tile tile;
    if (p.normalize) {
        tile.load(chunk_rows(p.q, w.n, w.hk, l0, Elem<T>::kBytes), (uint32_t)p.q.stride_l * Elem<T>::kBytes, p.E,
                  w.valid, p.vec_q, tid);
        squares(tile, (lds_float *)q2_mem, tid);
    }
    tile.load(chunk_rows(p.k, w.n, w.hk, l0, Elem<T>::kBytes), (uint32_t)p.k.stride_l * Elem<T>::kBytes, p.E, w.valid,
              p.vec_k, tid);
    if (p.normalize) squares(tile, (lds_float *)k2_mem, tid);
    tile.template store<RB>(kp, tid);
    __syncthreads();

    float *const factors = p.factors + w.at * (kFactors * kRows);
    if (wave == 0) {
        // the cumulative log decays in 64 bits: their differences are exponents.  (-1000 stands for everything
        // below: exp of it is zero, and sums of it stay finite.)
        double g = 0.0;
        float b = 0.f, back = 0.f;  // (beta, and as the backward has it)
        bool shut = false;
        if (lane < w.valid) {
            const int64_t l = l0 + lane;
            const float x = load_as_f32(p.g.ptr, p.g.dtype, w.n * p.g.sn + w.h * p.g.sh + l * p.g.sl);
            g = x < -1000.f ? -1000.0 : (double)x;
            b = load_as_f32(p.b.ptr, p.b.dtype, w.n * p.b.sn + w.h * p.b.sh + l * p.b.sl);
            shut = fabsf(b) <= kLeastBeta, back = shut ? kLeastBeta : b;
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double other = __shfl_up(g, d);
            if (lane >= d) g += other;
        }
        const double total = __shfl(g, 63);
        const float high = (float)g, low = (float)(g - (double)high);
        const float rk = p.normalize ? (float)(1.0 / sqrt((double)k2_mem[lane] + (double)kNormEps)) : 1.f;
        const float rq0 = p.normalize ? (float)(1.0 / sqrt((double)q2_mem[lane] + (double)kNormEps)) : 1.f;
        const float rise = (float)exp(g), fall = (float)exp(total - g);
        factors[kRise * kRows + lane] = rise;
        factors[kFall * kRows + lane] = fall;
        factors[kReadK * kRows + lane] = rk * rise;
        factors[kReadQ * kRows + lane] = rq0 * p.scale * rise;
        factors[kWriteK * kRows + lane] = rk * fall;
        factors[kWrite * kRows + lane] = rk * fall * b;
        factors[kBeta * kRows + lane] = b;
        factors[kRk * kRows + lane] = rk;
        factors[kRq * kRows + lane] = rq0 * p.scale;
        factors[kRq0 * kRows + lane] = rq0;
        factors[kHigh * kRows + lane] = high;
        factors[kLow * kRows + lane] = low;
        if (p.tt) {
            factors[kBetaBack * kRows + lane] = back;
            factors[kWriteBack * kRows + lane] = rk * fall * back;
            factors[kReadBack * kRows + lane] = shut ? 0.f : rk * rise;
            factors[kRkBack * kRows + lane] = shut ? 0.f : rk;
        }
        high_mem[lane] = high, low_mem[lane] = low, beta_mem[0][lane] = b, beta_mem[1][lane] = back, rk_mem[lane] = rk;
        again_mem = p.tt && __any(shut);
    }
    __syncthreads();

    // the keys' fragments, by the first value head of the key head
    if (w.h % (p.H / p.Hk) == 0) {
        uint16_t *const kr = p.kr + w.key_at * (4 * KE * PIECES * 512), *const kc = p.kc + w.key_at * (4 * KE * PIECES * 512);
        for (int i = wave; i < 4 * KE; i += 4) {
            Frag f[PIECES];
            rows_of<RB>(kp, i / KE, i % KE, c, q, f);
            store_frag(kr, i, lane, f);
            columns_of<RB>(kp, i / 2, i % 2, c, q, f);
            store_frag(kc, i, lane, f);
        }
    }

    // T, and where the backward has other betas a second time, for the transpose that it reads
    const bool again = scalar(again_mem) != 0;
    for (int turn = 0;; turn++) {
        asm volatile("" : "+v"(tid), "+v"(lane), "+v"(c), "+v"(q));  // (addresses of both turns, held at once, are registers)
        const float *const beta = beta_mem[turn];
        // M: the ten tiles on and below the diagonal
        for (int id = wave; id < 10; id += 4) {
            const int ti = id < 1 ? 0 : id < 3 ? 1 : id < 6 ? 2 : 3, tj = id - ti * (ti + 1) / 2;
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KE; s++) {
                Frag a[PIECES], b[PIECES];
                rows_of<RB>(kp, ti, s, c, q, a);
                rows_of<RB>(kp, tj, s, c, q, b);
                acc = product(a, b, acc);
            }
            const int j = 16 * tj + c;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = 16 * ti + 4 * q + r;
                const float d = expf((high_mem[i] - high_mem[j]) + (low_mem[i] - low_mem[j]));
                Mx[i * kStride + j] = j < i ? acc[r] * d * (rk_mem[i] * rk_mem[j]) * beta[j] : 0.f;
            }
        }
        __syncthreads();
        for (int i = tid; i < kRows * kStride; i += kThreads) Tm[i] = 0.f;
        __syncthreads();

        // diagonal blocks: column c of block `wave`
        if (lane < 16) {
            const lds_float *const m = Mx + 16 * wave * kStride + 16 * wave;
            float x[16];
#pragma unroll
            for (int r = 0; r < 16; r++) {
                float sum = r == lane ? 1.f : 0.f;
#pragma unroll
                for (int s = 0; s < r; s++) sum = fmaf(-m[r * kStride + s], x[s], sum);
                x[r] = sum;
            }
#pragma unroll
            for (int r = 0; r < 16; r++) Tm[(16 * wave + r) * kStride + 16 * wave + lane] = x[r];
        }
        __syncthreads();
        // blocks of 32: rows 16 (2 w + 1), columns 32 w, by wavefronts 0 and 1.  (Instruction r takes k = 4 q + r, the
        // order in which the first product's result lies in the registers.)
        if (wave < 2) {
            const int r0 = 32 * wave + 16, c0 = 32 * wave;
            f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < 4; r++)
                x = mfma_f32(Mx[(r0 + c) * kStride + c0 + 4 * q + r], Tm[(c0 + 4 * q + r) * kStride + c0 + c], x);
#pragma unroll
            for (int r = 0; r < 4; r++) y = mfma_f32(Tm[(r0 + c) * kStride + r0 + 4 * q + r], x[r], y);
#pragma unroll
            for (int r = 0; r < 4; r++) Tm[(r0 + 4 * q + r) * kStride + c0 + c] = -y[r];
        }
        __syncthreads();
        // the block of 64: a wavefront per tile
        {
            const int a = wave >> 1, b = wave & 1;
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    x = mfma_f32(Mx[(32 + 16 * a + c) * kStride + 16 * kt + 4 * q + r],
                                 Tm[(16 * kt + 4 * q + r) * kStride + 16 * b + c], x);
#pragma unroll
            for (int r = 0; r < 4; r++) X[(16 * a + 4 * q + r) * kStride + 16 * b + c] = x[r];
            __syncthreads();
            f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    y = mfma_f32(Tm[(32 + 16 * a + c) * kStride + 32 + 16 * kt + 4 * q + r],
                                 X[(16 * kt + 4 * q + r) * kStride + 16 * b + c], y);
#pragma unroll
            for (int r = 0; r < 4; r++) Tm[(32 + 16 * a + 4 * q + r) * kStride + 16 * b + c] = -y[r];
        }
        __syncthreads();
        // T in pieces where M was, and from there its fragments
        lds_char *const tp = (lds_char *)m_mem;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int u = tid + kThreads * i, row = u / 16, slot = u % 16;
            const lds_float *const x = Tm + row * kStride + 4 * slot;
            store_pieces(tp + Plane<128>::addr(row, slot), Plane<128>::kBytes, f32x4{x[0], x[1], x[2], x[3]});
        }
        __syncthreads();
        for (int i = wave; i < kTFrags; i += 4) {
            Frag f[3];
            const int t = i < 2 ? i : 1 + i / 2, s = i < 2 ? 0 : i % 2;
            rows_of<128>(tp, t, s, c, q, f);
            if (turn == 0) store_frag(p.t + w.at * (kTFrags * 3 * 512), i, lane, f);
            if (!p.tt || (again && turn == 0)) continue;
            const int u = i < 4 ? i / 2 : i - 2, v = i < 4 ? i % 2 : 1;
            columns_of<128>(tp, u, v, c, q, f);
            store_frag(p.tt + w.at * (kTFrags * 3 * 512), i, lane, f);
        }
        if (!again || turn == 1) return;
        __syncthreads();  // (T lay where k and M come now)
        tile.load(chunk_rows(p.k, w.n, w.hk, l0, Elem<T>::kBytes), (uint32_t)p.k.stride_l * Elem<T>::kBytes, p.E, w.valid,
                  p.vec_k, tid);
        tile.template store<RB>(kp, tid);
        __syncthreads();
    }
}

}  // namespace

int delta_prepare(const DeltaArgs &p, bool bf16, hipStream_t stream) {
    const dim3 grid((uint32_t)p.N * (uint32_t)p.H * (uint32_t)p.chunks);
    if (p.E <= 64) {
        if (bf16) delta_prepare_kernel<bf16_t, 2><<<grid, kThreads, 0, stream>>>(p);
        else delta_prepare_kernel<float, 2><<<grid, kThreads, 0, stream>>>(p);
    } else {
        if (bf16) delta_prepare_kernel<bf16_t, 4><<<grid, kThreads, 0, stream>>>(p);
        else delta_prepare_kernel<float, 4><<<grid, kThreads, 0, stream>>>(p);
    }
    return FTC_OK;
}

}  // namespace delta
}  // namespace ftc
