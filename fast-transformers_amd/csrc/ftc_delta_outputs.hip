// The gated delta rule, what the chunks compute from the states before them, all chunks side by side:
// the outputs O = diag(rq e^G) Q S + A diag(beta) Z and, for the backward, A^T dO and dO . O.  Formulas and layouts:
// ftc_delta_kernel.h.
//
// A workgroup of four wavefronts takes one chunk and 16 CT columns per wavefront: A once for all of them, in LDS in
// three pieces, then a wavefront's columns of the products.
//
// What bounds it: memory where there are many chunks.  A lies where k was (and q, in A^T dO), so that four and five workgroups
// fit a compute unit (bf16); results are stored four columns a lane.  Measured: 8192 chunks of 128 x 128, bf16: outputs 320 us, 4.2 TB/s
// of states, Z, rows, out and O (two workgroups a compute unit, and a value a store: 410); A^T dO 181 us, 4.9 TB/s
// (243).  1280 chunks of 64 x 64, fp32: 32 and 35 us.
#include "ftc_delta_kernel.h"
#include <type_traits>

namespace ftc {
namespace delta {
namespace {

constexpr int kThreads = 256;
constexpr int kAPlane = Plane<128>::kBytes;

// A wavefront's three tiles of A.  Its transpose is what is multiplied, so that a lane has four consecutive
// columns.  The tiles above the diagonal that share a k-step with it are zero.
struct TilesOfA {
    f32x4 x[3];
    __device__ static __forceinline__ int row_tile(int id) { return id < 2 ? 0 : id < 4 ? 1 : id < 8 ? 2 : 3; }
    __device__ static __forceinline__ int column_tile(int id) { return id < 4 ? id & 1 : id & 3; }
    template <int RB, int KE, int PIECES>
    __device__ __forceinline__ void make(const lds_char *qp, const lds_char *kp, const float *factors, int wave, int c, int q) {
#pragma unroll
        for (int n = 0; n < 3; n++) {
            const int ti = row_tile(wave + 4 * n), tj = column_tile(wave + 4 * n);
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
                x[n][r] = j0 + r <= i ? acc[r] * expf((high_i - high[r]) + (low_i - low[r])) * (rq * rk[r]) : 0.f;
        }
    }
    // to three planes, row i, column j
    __device__ __forceinline__ void put(lds_char *ap, int wave, int c, int q) const {
#pragma unroll
        for (int n = 0; n < 3; n++)
            store_pieces(ap + Plane<128>::addr(16 * row_tile(wave + 4 * n) + c, 4 * column_tile(wave + 4 * n) + q), kAPlane, x[n]);
    }
};

// Rows of q and k into LDS
template <typename T, int KE>
__device__ __forceinline__ void stage(const DeltaArgs &p, const Where &w, lds_char *qp, lds_char *kp, int tid) {
    constexpr int RB = 64 * KE;
    RowTile<T, 32 * KE, kThreads> q_tile, k_tile;
    const int64_t l0 = (int64_t)w.chunk * kRows;
    q_tile.load(chunk_rows(p.q, w.n, w.hk, l0, Elem<T>::kBytes), (uint32_t)p.q.stride_l * Elem<T>::kBytes, p.E, w.valid,
                p.vec_q, tid);
    k_tile.load(chunk_rows(p.k, w.n, w.hk, l0, Elem<T>::kBytes), (uint32_t)p.k.stride_l * Elem<T>::kBytes, p.E, w.valid,
                p.vec_k, tid);
    q_tile.template store<RB>(qp, tid);
    k_tile.template store<RB>(kp, tid);
    __syncthreads();
}
// Four lanes side by side exchange: lane j of them has value j of all four
__device__ __forceinline__ void exchange(f32x4 &x, int lane) {
    auto beside = [](float v, auto control) {
        return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), decltype(control)::value, 0xf, 0xf, false));
    };
    const bool odd = lane & 1, high = lane & 2;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const float there = beside(odd ? x[i] : x[i + 1], std::integral_constant<int, 0xb1>());  // lanes 1 0 3 2
        x[i] = odd ? there : x[i], x[i + 1] = odd ? x[i + 1] : there;
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float there = beside(high ? x[i] : x[i + 2], std::integral_constant<int, 0x4e>());  // lanes 2 3 0 1
        x[i] = high ? there : x[i], x[i + 2] = high ? x[i + 2] : there;
    }
}

template <typename T, int KE, int CT>
__global__ __launch_bounds__(kThreads) void delta_outputs_kernel(DeltaArgs p) {
    constexpr int RB = 64 * KE, PIECES = Elem<T>::kPieces, ET = 2 * KE;
    constexpr int kPlanes = PIECES * Plane<RB>::kBytes;
    // (A where k was)
    __shared__ __align__(16) char q_mem[kPlanes], k_mem[kPlanes > 3 * kAPlane ? kPlanes : 3 * kAPlane];
    lds_char *const qp = (lds_char *)q_mem, *const kp = (lds_char *)k_mem, *const ap = kp;
    const int tid = threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6), c = lane & 15, q = lane >> 4;
    const int groups = (p.col_blocks + 4 * CT - 1) / (4 * CT);
    const uint32_t id = blockIdx.x / (uint32_t)groups;
    const int first = (int)(blockIdx.x % (uint32_t)groups) * 4 * CT + wave * CT;
    const Where w = where_of(p, (int)(id / (uint32_t)p.chunks), (int)(id % (uint32_t)p.chunks));
    const float *const factors = p.factors + w.at * (kFactors * kRows);
    const int64_t l0 = (int64_t)w.chunk * kRows;
    const int rows = min((int64_t)kRows, p.L - l0);
    const int64_t out0 = w.n * p.out.stride_n + w.h * p.out.stride_h + l0 * p.out.stride_l;
    if (w.valid > 0) {
        TilesOfA A;
        stage<T, KE>(p, w, qp, kp, tid);
        A.make<RB, KE, PIECES>(qp, kp, factors, wave, c, q);
        __syncthreads();
        A.put(ap, wave, c, q);
        __syncthreads();
    }

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
        if (p.vec_out) {  // four columns of a row a lane
#pragma unroll
            for (int t = 0; t < 4; t++) {
                exchange(O[t], lane);
                const int row = 16 * t + 4 * q + (c & 3), at = kCols * block + (c & ~3);
                if (row >= rows || at >= p.M) continue;
                T *const to = (T *)p.out.ptr + out0 + row * p.out.stride_l + at;
                if constexpr (Elem<T>::kBytes == 4) {
                    *(f32x4a *)to = O[t];
                } else {
                    *(u32x2a *)to = u32x2{to_bf16(O[t][0], O[t][1]), to_bf16(O[t][2], O[t][3])};
                }
            }
        } else if (col < p.M)
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
    constexpr int kPlanes = PIECES * Plane<RB>::kBytes;
    // (A where q and k were)
    __shared__ __align__(16) char mem[2 * kPlanes > 3 * kAPlane ? 2 * kPlanes : 3 * kAPlane];
    lds_char *const qp = (lds_char *)mem, *const kp = qp + kPlanes, *const ap = qp;
    const int tid = threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6), c = lane & 15, q = lane >> 4;
    const int groups = (p.col_blocks + 4 * CT - 1) / (4 * CT);
    const uint32_t id = blockIdx.x / (uint32_t)groups;
    const int first = (int)(blockIdx.x % (uint32_t)groups) * 4 * CT + wave * CT;
    const Where w = where_of(p, (int)(id / (uint32_t)p.chunks), (int)(id % (uint32_t)p.chunks));
    const float *const factors = p.factors + w.at * (kFactors * kRows);
    if (w.valid == 0) return;
    stage<T, KE>(p, w, qp, kp, tid);
    TilesOfA A;
    A.make<RB, KE, PIECES>(qp, kp, factors, wave, c, q);
    // the queries' fragments, by the first workgroup of the first value head
    if (w.h % (p.H / p.Hk) == 0 && blockIdx.x % (uint32_t)groups == 0)
        for (int i = wave; i < 4 * KE; i += 4) {
            Frag f[PIECES];
            columns_of<RB>(qp, i / 2, i % 2, c, q, f);
            store_frag(p.qc + w.key_at * (4 * KE * PIECES * 512), i, lane, f);
        }
    __syncthreads();
    A.put(ap, wave, c, q);
    __syncthreads();

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
