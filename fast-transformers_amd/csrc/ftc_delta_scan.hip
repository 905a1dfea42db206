// The gated delta rule's state from chunk to chunk, forward (Z of every position, the state before every chunk and
// after the last) and backward (the gradient of the state, dE = dV).  Formulas and layouts: ftc_delta_kernel.h.
//
// A wavefront owns 16 columns of one chain's state in registers and walks the chunks; what it multiplies with, the
// rows of k (and q) and T, the workgroup stages in LDS, each chunk's while the one before is worked on.
#include "ftc_delta_kernel.h"

namespace ftc {
namespace delta {
namespace {

constexpr int kTPlane = Plane<128>::kBytes;
constexpr int kFactorFloats = kFactors * kRows;

// T of a chunk: 3 planes of 64 x 64, into registers and on into LDS
template <int NT>
struct TTile {
    static constexpr int kPer = 3 * kRows * 8 / NT;
    u32x4 r[kPer];
    __device__ __forceinline__ void load(const uint16_t *t, int tid) {
#pragma unroll
        for (int i = 0; i < kPer; i++) r[i] = *(const u32x4a *)(t + 8 * (tid + NT * i));
    }
    __device__ __forceinline__ void store(lds_char *planes, int tid) const {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int u = tid + NT * i, piece = u / (kRows * 8), row = (u / 8) % kRows;
            *(__attribute__((address_space(3))) u32x4a *)(planes + piece * kTPlane + Plane<128>::addr(row, 2 * (u % 8))) =
                r[i];
        }
    }
};
template <int NT>
struct FactorTile {
    static constexpr int kPer = (kFactorFloats / 4 + NT - 1) / NT;
    f32x4 r[kPer];
    __device__ __forceinline__ void load(const float *f, int tid) {
#pragma unroll
        for (int i = 0; i < kPer; i++)
            if (tid + NT * i < kFactorFloats / 4) r[i] = *(const f32x4a *)(f + 4 * (tid + NT * i));
    }
    __device__ __forceinline__ void store(lds_float *to, int tid) const {
#pragma unroll
        for (int i = 0; i < kPer; i++)
            if (tid + NT * i < kFactorFloats / 4)
                *(__attribute__((address_space(3))) f32x4a *)(to + 4 * (tid + NT * i)) = r[i];
    }
};
// rows 16 t + 4 q .. of a factor
__device__ __forceinline__ f32x4 factor(const lds_float *f, int which, int t, int q) {
    return *(const __attribute__((address_space(3))) f32x4a *)(f + which * kRows + 16 * t + 4 * q);
}

// Values of rows 16 t + 4 q + r of a column
template <typename T>
__device__ __forceinline__ void load_column(__amdgpu_buffer_rsrc_t rs, uint32_t row_bytes, int col, int width, int valid,
                                            int q, f32x4 (&x)[4]) {
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = 16 * t + 4 * q + r;
            x[t][r] = load_one<T>(rs, row < valid && col < width ? (uint32_t)row * row_bytes + (uint32_t)(col * Elem<T>::kBytes)
                                                                 : kOutside);
        }
}

template <typename T, int KE, int NW>
__global__ __launch_bounds__(64 * NW) void delta_scan_kernel(DeltaArgs p) {
    constexpr int NT = 64 * NW, RB = 64 * KE, PIECES = Elem<T>::kPieces, ET = 2 * KE;
    __shared__ __align__(16) char k_mem[PIECES * Plane<RB>::kBytes], t_mem[3 * kTPlane];
    __shared__ __align__(16) float f_mem[kFactorFloats];
    lds_char *const kp = (lds_char *)k_mem, *const tp = (lds_char *)t_mem;
    lds_float *const fp = (lds_float *)f_mem;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
    const int groups = (p.col_blocks + NW - 1) / NW;
    const int block = (int)(blockIdx.x % (uint32_t)groups) * NW + wave, col = kCols * block + c;
    const Where w = where_of(p, (int)(blockIdx.x / (uint32_t)groups), 0);
    const int chunks = chunks_of(w.len);
    const bool mine = block < p.col_blocks;

    f32x4 S[ET];
#pragma unroll
    for (int t = 0; t < ET; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int e = 16 * t + 4 * q + r;
            S[t][r] = p.initial.ptr && e < p.E && col < p.M
                          ? p.initial.ptr[w.n * p.initial.stride_n + w.h * p.initial.stride_h + e * p.initial.stride_d + col]
                          : 0.f;
        }

    RowTile<T, 32 * KE, NT> k_tile;
    TTile<NT> t_tile;
    FactorTile<NT> f_tile;
    f32x4 V[4];
    const uint32_t k_row = (uint32_t)p.k.stride_l * Elem<T>::kBytes, v_row = (uint32_t)p.v.stride_l * Elem<T>::kBytes;
    auto request = [&](int chunk) {
        const int64_t at = (int64_t)w.chain * p.chunks + chunk, l0 = (int64_t)chunk * kRows;
        const int valid = min(kRows, w.len - chunk * kRows);
        k_tile.load(chunk_rows(p.k, w.n, w.hk, l0, Elem<T>::kBytes), k_row, p.E, valid, p.vec_k, tid);
        t_tile.load(p.t + at * (3 * kRows * kRows), tid);
        f_tile.load(p.factors + at * kFactorFloats, tid);
        load_column<T>(chunk_rows(p.v, w.n, w.h, l0, Elem<T>::kBytes), v_row, col, p.M, valid, q, V);
    };
    if (chunks > 0) request(0);
    for (int chunk = 0; chunk < chunks; chunk++) {
        const int64_t at = (int64_t)w.chain * p.chunks + chunk;
        __syncthreads();
        k_tile.template store<RB>(kp, tid);
        t_tile.store(tp, tid);
        f_tile.store(fp, tid);
        f32x4 Z[4];
#pragma unroll
        for (int t = 0; t < 4; t++) Z[t] = V[t];
        __syncthreads();
        if (chunk + 1 < chunks) request(chunk + 1);

        if (p.s && mine) {
            float *const to = p.s + (at * p.col_blocks + block) * (ET * 256) + 4 * lane;
#pragma unroll
            for (int t = 0; t < ET; t++) *(f32x4a *)(to + 256 * t) = S[t];
        }
        // E = V - diag(rk e^G) K S
        f32x4 P[4] = {};
#pragma unroll
        for (int s = 0; s < KE; s++) {
            Frag sf[3];
            cut(S[2 * s], S[2 * s + 1], sf);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                Frag kf[PIECES];
                rows_of<RB>(kp, t, s, c, q, kf);
                P[t] = product(kf, sf, P[t]);
            }
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const f32x4 f = factor(fp, kRise, t, q) * factor(fp, kRk, t, q);
            P[t] = Z[t] - f * P[t];
            Z[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        // Z = T E (tiles above the diagonal are zero)
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag ef[3];
            cut(P[2 * s], P[2 * s + 1], ef);
#pragma unroll
            for (int t = 2 * s; t < 4; t++) {
                Frag tf[3];
                rows_of<128>(tp, t, s, c, q, tf);
                Z[t] = product(tf, ef, Z[t]);
            }
        }
        if (p.z && mine) {
            float *const to = p.z + (at * p.col_blocks + block) * (4 * 256) + 4 * lane;
#pragma unroll
            for (int t = 0; t < 4; t++) *(f32x4a *)(to + 256 * t) = Z[t];
        }
        // S <- e^{G_64} S + K^T diag(rk beta e^{G_64 - G}) Z
        const float last = fp[kRise * kRows + kRows - 1];
#pragma unroll
        for (int t = 0; t < 4; t++) Z[t] *= factor(fp, kFall, t, q) * factor(fp, kBeta, t, q) * factor(fp, kRk, t, q);
#pragma unroll
        for (int t = 0; t < ET; t++) S[t] *= last;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag uf[3];
            cut(Z[2 * s], Z[2 * s + 1], uf);
#pragma unroll
            for (int t = 0; t < ET; t++) {
                Frag kf[PIECES];
                columns_of<RB>(kp, t, s, c, q, kf);
                S[t] = product(kf, uf, S[t]);
            }
        }
    }
    if (p.final_.ptr && mine)
#pragma unroll
        for (int t = 0; t < ET; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int e = 16 * t + 4 * q + r;
                if (e < p.E && col < p.M)
                    p.final_.ptr[w.n * p.final_.stride_n + w.h * p.final_.stride_h + e * p.final_.stride_d + col] = S[t][r];
            }
}

// The same walk from the last chunk to the first, on the gradient of the state:
//   dU = A^T dO + diag(rk e^{G_64 - G}) K dS,   dE = T^T diag(beta) dU,
//   dS <- e^{G_64} dS + Q^T diag(rq e^G) dO - K^T diag(rk e^G) dE
template <typename T, int KE, int NW>
__global__ __launch_bounds__(64 * NW) void delta_scan_back_kernel(DeltaArgs p) {
    constexpr int NT = 64 * NW, RB = 64 * KE, PIECES = Elem<T>::kPieces, ET = 2 * KE;
    __shared__ __align__(16) char k_mem[PIECES * Plane<RB>::kBytes], q_mem[PIECES * Plane<RB>::kBytes], t_mem[3 * kTPlane];
    __shared__ __align__(16) float f_mem[kFactorFloats];
    lds_char *const kp = (lds_char *)k_mem, *const qp = (lds_char *)q_mem, *const tp = (lds_char *)t_mem;
    lds_float *const fp = (lds_float *)f_mem;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
    const int groups = (p.col_blocks + NW - 1) / NW;
    const int block = (int)(blockIdx.x % (uint32_t)groups) * NW + wave, col = kCols * block + c;
    const Where w = where_of(p, (int)(blockIdx.x / (uint32_t)groups), 0);
    const int chunks = chunks_of(w.len);
    const bool mine = block < p.col_blocks;

    f32x4 S[ET];
#pragma unroll
    for (int t = 0; t < ET; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int e = 16 * t + 4 * q + r;
            S[t][r] = p.grad_final.ptr && e < p.E && col < p.M
                          ? p.grad_final.ptr[w.n * p.grad_final.stride_n + w.h * p.grad_final.stride_h +
                                             e * p.grad_final.stride_d + col]
                          : 0.f;
        }

    RowTile<T, 32 * KE, NT> k_tile, q_tile;
    TTile<NT> t_tile;
    FactorTile<NT> f_tile;
    f32x4 G[4], Y[4], Zn[4];
    const uint32_t k_row = (uint32_t)p.k.stride_l * Elem<T>::kBytes, q_row = (uint32_t)p.q.stride_l * Elem<T>::kBytes,
                   g_row = (uint32_t)p.go.stride_l * Elem<T>::kBytes;
    auto request = [&](int chunk) {
        const int64_t at = (int64_t)w.chain * p.chunks + chunk, l0 = (int64_t)chunk * kRows;
        const int valid = min(kRows, w.len - chunk * kRows);
        k_tile.load(chunk_rows(p.k, w.n, w.hk, l0, Elem<T>::kBytes), k_row, p.E, valid, p.vec_k, tid);
        q_tile.load(chunk_rows(p.q, w.n, w.hk, l0, Elem<T>::kBytes), q_row, p.E, valid, p.vec_q, tid);
        t_tile.load(p.t + at * (3 * kRows * kRows), tid);
        f_tile.load(p.factors + at * kFactorFloats, tid);
        load_column<T>(chunk_rows(p.go, w.n, w.h, l0, Elem<T>::kBytes), g_row, col, p.M, valid, q, G);
        if (mine) {
            const int64_t z = (at * p.col_blocks + block) * (4 * 256) + 4 * lane;
#pragma unroll
            for (int t = 0; t < 4; t++) Y[t] = *(const f32x4a *)(p.de + z + 256 * t);
#pragma unroll
            for (int t = 0; t < 4; t++) Zn[t] = *(const f32x4a *)(p.z + z + 256 * t);
        }
    };
#pragma unroll
    for (int t = 0; t < 4; t++) Y[t] = Zn[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (chunks > 0) request(chunks - 1);
    for (int chunk = chunks - 1; chunk >= 0; chunk--) {
        const int64_t at = (int64_t)w.chain * p.chunks + chunk;
        const int valid = min(kRows, w.len - chunk * kRows);
        __syncthreads();
        k_tile.template store<RB>(kp, tid);
        q_tile.template store<RB>(qp, tid);
        t_tile.store(tp, tid);
        f_tile.store(fp, tid);
        f32x4 D[4], Z[4], O[4];
#pragma unroll
        for (int t = 0; t < 4; t++) D[t] = Y[t], Z[t] = Zn[t], O[t] = G[t];
        __syncthreads();
        if (chunk > 0) request(chunk - 1);

        if (mine) {
            float *const to = p.ds + (at * p.col_blocks + block) * (ET * 256) + 4 * lane;
#pragma unroll
            for (int t = 0; t < ET; t++) *(f32x4a *)(to + 256 * t) = S[t];
        }
        f32x4 P[4] = {};
#pragma unroll
        for (int s = 0; s < KE; s++) {
            Frag sf[3];
            cut(S[2 * s], S[2 * s + 1], sf);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                Frag kf[PIECES];
                rows_of<RB>(kp, t, s, c, q, kf);
                P[t] = product(kf, sf, P[t]);
            }
        }
        // dU, its products with Z (the gradient of beta), and diag(beta) dU
#pragma unroll
        for (int t = 0; t < 4; t++) {
            D[t] += factor(fp, kFall, t, q) * factor(fp, kRk, t, q) * P[t];
            f32x4 dot = Z[t] * D[t];
#pragma unroll
            for (int r = 0; r < 4; r++) dot[r] = sum16(dot[r]);
            if (mine && c == 0) *(f32x4a *)(p.zdu + (at * p.col_blocks + block) * kRows + 16 * t + 4 * q) = dot;
            D[t] *= factor(fp, kBeta, t, q);
            P[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        // dE = T^T diag(beta) dU
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag df[3];
            cut(D[2 * s], D[2 * s + 1], df);
#pragma unroll
            for (int t = 0; t < 2 * s + 2; t++) {
                Frag tf[3];
                columns_of<128>(tp, t, s, c, q, tf);
                P[t] = product(tf, df, P[t]);
            }
        }
        if (mine) {
            float *const to = p.de + (at * p.col_blocks + block) * (4 * 256) + 4 * lane;
#pragma unroll
            for (int t = 0; t < 4; t++) *(f32x4a *)(to + 256 * t) = P[t];
            if (p.gv.ptr && col < p.M)
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int row = 16 * t + 4 * q + r;
                        if (row < valid)
                            store_from_f32(p.gv.ptr, p.gv.dtype,
                                           w.n * p.gv.stride_n + w.h * p.gv.stride_h +
                                               ((int64_t)chunk * kRows + row) * p.gv.stride_l + col, P[t][r]);
                    }
        }
        const float last = fp[kRise * kRows + kRows - 1];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const f32x4 rise = factor(fp, kRise, t, q);
            O[t] *= rise * factor(fp, kRq, t, q);
            P[t] *= -rise * factor(fp, kRk, t, q);
        }
#pragma unroll
        for (int t = 0; t < ET; t++) S[t] *= last;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag of[3], ef[3];
            cut(O[2 * s], O[2 * s + 1], of);
            cut(P[2 * s], P[2 * s + 1], ef);
#pragma unroll
            for (int t = 0; t < ET; t++) {
                Frag f[PIECES];
                columns_of<RB>(qp, t, s, c, q, f);
                S[t] = product(f, of, S[t]);
                columns_of<RB>(kp, t, s, c, q, f);
                S[t] = product(f, ef, S[t]);
            }
        }
    }
    if (!mine) return;
    if (p.grad_initial.ptr)
#pragma unroll
        for (int t = 0; t < ET; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int e = 16 * t + 4 * q + r;
                if (e < p.E && col < p.M)
                    p.grad_initial.ptr[w.n * p.grad_initial.stride_n + w.h * p.grad_initial.stride_h +
                                       e * p.grad_initial.stride_d + col] = S[t][r];
            }
    // positions past the end of the sequence
    if (p.gv.ptr && col < p.M)
        for (int l = w.len + q; l < p.L; l += 4)
            store_from_f32(p.gv.ptr, p.gv.dtype, w.n * p.gv.stride_n + w.h * p.gv.stride_h + l * p.gv.stride_l + col, 0.f);
}

template <typename T, int KE>
void launch(const DeltaArgs &p, bool back, hipStream_t stream) {
    constexpr int NW = 4;
    const dim3 grid((uint32_t)p.N * (uint32_t)p.H * (uint32_t)((p.col_blocks + NW - 1) / NW));
    if (back) delta_scan_back_kernel<T, KE, NW><<<grid, 64 * NW, 0, stream>>>(p);
    else delta_scan_kernel<T, KE, NW><<<grid, 64 * NW, 0, stream>>>(p);
}
int dispatch(const DeltaArgs &p, bool bf16, bool back, hipStream_t stream) {
    if (p.E <= 64) bf16 ? launch<bf16_t, 2>(p, back, stream) : launch<float, 2>(p, back, stream);
    else bf16 ? launch<bf16_t, 4>(p, back, stream) : launch<float, 4>(p, back, stream);
    return FTC_OK;
}

}  // namespace

int delta_scan(const DeltaArgs &p, bool bf16, hipStream_t stream) { return dispatch(p, bf16, false, stream); }
int delta_scan_back(const DeltaArgs &p, bool bf16, hipStream_t stream) { return dispatch(p, bf16, true, stream); }

}  // namespace delta
}  // namespace ftc
