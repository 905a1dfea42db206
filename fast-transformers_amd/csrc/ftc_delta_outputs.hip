// The gated delta rule, what the chunks compute from the states before them, all chunks side by side:
// the outputs O = diag(rq e^G) Q S + A diag(beta) Z and, for the backward, A^T dO and dO . O.  Formulas and layouts:
// ftc_delta_kernel.h.
//
// A workgroup of four wavefronts takes one chunk and 16 CT columns per wavefront: A once for all of them, in LDS in
// three pieces, then a wavefront's columns of the products.
#include "ftc_delta_kernel.h"

namespace ftc {
namespace delta {
namespace {

constexpr int kThreads = 256;
constexpr int kAPlane = Plane<128>::kBytes;

// A to three planes (row i, column j).  Its transpose is what is multiplied, so that a lane has four
// consecutive columns.  The tiles above the diagonal that share a k-step with it are zero.
template <int RB, int KE, int PIECES>
__device__ __forceinline__ void make_a(const lds_char *qp, const lds_char *kp, lds_char *ap, const float *factors,
                                       int wave, int c, int q) {
#pragma unroll
    for (int x = 0; x < 3; x++) {
        const int id = wave + 4 * x, ti = id < 2 ? 0 : id < 4 ? 1 : id < 8 ? 2 : 3,
                  tj = id < 4 ? id & 1 : id & 3;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KE; s++) {
            Frag a[PIECES], b[PIECES];
            rows_of<RB>(kp, tj, s, c, q, a);
            rows_of<RB>(qp, ti, s, c, q, b);
            acc = product(a, b, acc);
        }
        const int i = 16 * ti + c, j0 = 16 * tj + 4 * q;
        const f32x4 high = *(const f32x4a *)(factors + kHigh * kRows + j0), low = *(const f32x4a *)(factors + kLow * kRows + j0),
                    rk = *(const f32x4a *)(factors + kRk * kRows + j0);
        const float high_i = factors[kHigh * kRows + i], low_i = factors[kLow * kRows + i], rq = factors[kRq * kRows + i];
#pragma unroll
        for (int r = 0; r < 4; r++)
            acc[r] = j0 + r <= i ? acc[r] * expf((high_i - high[r]) + (low_i - low[r])) * (rq * rk[r]) : 0.f;
        store_pieces(ap + Plane<128>::addr(i, 4 * tj + q), kAPlane, acc);
    }
}

// Rows of q and k into LDS, and A from them
template <typename T, int KE>
__device__ __forceinline__ void stage(const DeltaArgs &p, const Where &w, const float *factors, lds_char *qp, lds_char *kp,
                                      lds_char *ap, int tid) {
    constexpr int RB = 64 * KE, PIECES = Elem<T>::kPieces;
    RowTile<T, 32 * KE, kThreads> q_tile, k_tile;
    const int64_t l0 = (int64_t)w.chunk * kRows;
    q_tile.load(chunk_rows(p.q, w.n, w.hk, l0, Elem<T>::kBytes), (uint32_t)p.q.stride_l * Elem<T>::kBytes, p.E, w.valid,
                p.vec_q, tid);
    k_tile.load(chunk_rows(p.k, w.n, w.hk, l0, Elem<T>::kBytes), (uint32_t)p.k.stride_l * Elem<T>::kBytes, p.E, w.valid,
                p.vec_k, tid);
    q_tile.template store<RB>(qp, tid);
    k_tile.template store<RB>(kp, tid);
    __syncthreads();
    make_a<RB, KE, PIECES>(qp, kp, ap, factors, tid >> 6, tid & 15, (tid & 63) >> 4);
    __syncthreads();
}

template <typename T, int KE, int CT>
__global__ __launch_bounds__(kThreads) void delta_outputs_kernel(DeltaArgs p) {
    constexpr int RB = 64 * KE, PIECES = Elem<T>::kPieces, ET = 2 * KE;
    __shared__ __align__(16) char q_mem[PIECES * Plane<RB>::kBytes], k_mem[PIECES * Plane<RB>::kBytes], a_mem[3 * kAPlane];
    lds_char *const qp = (lds_char *)q_mem, *const kp = (lds_char *)k_mem, *const ap = (lds_char *)a_mem;
    const int tid = threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6), c = lane & 15, q = lane >> 4;
    const int groups = (p.col_blocks + 4 * CT - 1) / (4 * CT);
    const uint32_t id = blockIdx.x / (uint32_t)groups;
    const int first = (int)(blockIdx.x % (uint32_t)groups) * 4 * CT + wave * CT;
    const Where w = where_of(p, (int)(id / (uint32_t)p.chunks), (int)(id % (uint32_t)p.chunks));
    const float *const factors = p.factors + w.at * (kFactors * kRows);
    const int64_t l0 = (int64_t)w.chunk * kRows;
    const int rows = min((int64_t)kRows, p.L - l0);
    const int64_t out0 = w.n * p.out.stride_n + w.h * p.out.stride_h + l0 * p.out.stride_l;
    if (w.valid > 0) stage<T, KE>(p, w, factors, qp, kp, ap, tid);

#pragma unroll
    for (int x = 0; x < CT; x++) {
        const int block = first + x, col = kCols * block + c;
        if (block >= p.col_blocks) break;
        f32x4 O[4] = {};
        if (w.valid > 0) {
            const float *const sp = p.s + (w.at * p.col_blocks + block) * (ET * 256) + 4 * lane;
            const float *const zp = p.z + (w.at * p.col_blocks + block) * (4 * 256) + 4 * lane;
            f32x4 S[ET], Z[4];
#pragma unroll
            for (int t = 0; t < ET; t++) S[t] = *(const f32x4a *)(sp + 256 * t);
#pragma unroll
            for (int t = 0; t < 4; t++) Z[t] = *(const f32x4a *)(zp + 256 * t);
#pragma unroll
            for (int s = 0; s < KE; s++) {
                Frag sf[3];
                cut(S[2 * s], S[2 * s + 1], sf);
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    Frag qf[PIECES];
                    rows_of<RB>(qp, t, s, c, q, qf);
                    O[t] = product(qf, sf, O[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int i0 = 16 * t + 4 * q;
                O[t] *= *(const f32x4a *)(factors + kReadQ * kRows + i0);
                Z[t] *= *(const f32x4a *)(factors + kBeta * kRows + i0);
            }
#pragma unroll
            for (int s = 0; s < 2; s++) {
                Frag uf[3];
                cut(Z[2 * s], Z[2 * s + 1], uf);
#pragma unroll
                for (int t = 2 * s; t < 4; t++) {
                    Frag af[3];
                    rows_of<128>(ap, t, s, c, q, af);
                    O[t] = product(af, uf, O[t]);
                }
            }
            settle();
            if (p.o) {
                float *const to = p.o + (w.at * p.col_blocks + block) * (4 * 256) + 4 * lane;
#pragma unroll
                for (int t = 0; t < 4; t++) *(f32x4a *)(to + 256 * t) = O[t];
            }
        }
        if (col < p.M)
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int row = 16 * t + 4 * q + r;
                    if (row < rows) store_from_f32(p.out.ptr, p.out.dtype, out0 + row * p.out.stride_l + col, O[t][r]);
                }
    }
}

template <typename T, int KE, int CT>
__global__ __launch_bounds__(kThreads) void delta_pull_kernel(DeltaArgs p) {
    constexpr int RB = 64 * KE, PIECES = Elem<T>::kPieces;
    __shared__ __align__(16) char q_mem[PIECES * Plane<RB>::kBytes], k_mem[PIECES * Plane<RB>::kBytes], a_mem[3 * kAPlane];
    lds_char *const qp = (lds_char *)q_mem, *const kp = (lds_char *)k_mem, *const ap = (lds_char *)a_mem;
    const int tid = threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6), c = lane & 15, q = lane >> 4;
    const int groups = (p.col_blocks + 4 * CT - 1) / (4 * CT);
    const uint32_t id = blockIdx.x / (uint32_t)groups;
    const int first = (int)(blockIdx.x % (uint32_t)groups) * 4 * CT + wave * CT;
    const Where w = where_of(p, (int)(id / (uint32_t)p.chunks), (int)(id % (uint32_t)p.chunks));
    const float *const factors = p.factors + w.at * (kFactors * kRows);
    if (w.valid == 0) return;
    stage<T, KE>(p, w, factors, qp, kp, ap, tid);
    // the queries' fragments, by the first workgroup of the first value head
    if (w.h % (p.H / p.Hk) == 0 && blockIdx.x % (uint32_t)groups == 0)
        for (int i = wave; i < 4 * KE; i += 4) {
            Frag f[PIECES];
            columns_of<RB>(qp, i / 2, i % 2, c, q, f);
            store_frag(p.qc + w.key_at * (4 * KE * PIECES * 512), i, lane, f);
        }

    const __amdgpu_buffer_rsrc_t rows = chunk_rows(p.go, w.n, w.h, (int64_t)w.chunk * kRows, Elem<T>::kBytes);
    const uint32_t row_bytes = (uint32_t)p.go.stride_l * Elem<T>::kBytes;
#pragma unroll
    for (int x = 0; x < CT; x++) {
        const int block = first + x, col = kCols * block + c;
        if (block >= p.col_blocks) break;
        f32x4 G[4], Y[4] = {};
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * t + 4 * q + r;
                G[t][r] = load_one<T>(rows, row < w.valid && col < p.M
                                                ? (uint32_t)row * row_bytes + (uint32_t)(col * Elem<T>::kBytes) : kOutside);
            }
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag gf[PIECES];
            cut(G[2 * s], G[2 * s + 1], gf);
#pragma unroll
            for (int t = 0; t < 2 * s + 2; t++) {
                Frag af[3];
                columns_of<128>(ap, t, s, c, q, af);
                Y[t] = product(af, gf, Y[t]);
            }
        }
        const int64_t at = w.at * p.col_blocks + block;
#pragma unroll
        for (int t = 0; t < 4; t++) *(f32x4a *)(p.de + at * (4 * 256) + 4 * lane + 256 * t) = Y[t];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            f32x4 dot = G[t] * *(const f32x4a *)(p.o + at * (4 * 256) + 4 * lane + 256 * t);
#pragma unroll
            for (int r = 0; r < 4; r++) dot[r] = sum16(dot[r]);
            if (c == 0) *(f32x4a *)(p.dots + at * kRows + 16 * t + 4 * q) = dot;
        }
    }
}

template <typename T, int KE>
void launch(const DeltaArgs &p, bool pull, hipStream_t stream) {
    // a wavefront takes two blocks of 16 columns where there are more than four
    const int ct = p.col_blocks > 4 ? 2 : 1, groups = (p.col_blocks + 4 * ct - 1) / (4 * ct);
    const dim3 grid((uint32_t)p.N * (uint32_t)p.H * (uint32_t)p.chunks * (uint32_t)groups);
    if (pull) {
        if (ct == 2) delta_pull_kernel<T, KE, 2><<<grid, kThreads, 0, stream>>>(p);
        else delta_pull_kernel<T, KE, 1><<<grid, kThreads, 0, stream>>>(p);
    } else {
        if (ct == 2) delta_outputs_kernel<T, KE, 2><<<grid, kThreads, 0, stream>>>(p);
        else delta_outputs_kernel<T, KE, 1><<<grid, kThreads, 0, stream>>>(p);
    }
}
int dispatch(const DeltaArgs &p, bool bf16, bool pull, hipStream_t stream) {
    if (p.E <= 64) bf16 ? launch<bf16_t, 2>(p, pull, stream) : launch<float, 2>(p, pull, stream);
    else bf16 ? launch<bf16_t, 4>(p, pull, stream) : launch<float, 4>(p, pull, stream);
    return FTC_OK;
}

}  // namespace

int delta_outputs(const DeltaArgs &p, bool bf16, hipStream_t stream) { return dispatch(p, bf16, false, stream); }
int delta_pull(const DeltaArgs &p, bool bf16, hipStream_t stream) { return dispatch(p, bf16, true, stream); }

}  // namespace delta
}  // namespace ftc
