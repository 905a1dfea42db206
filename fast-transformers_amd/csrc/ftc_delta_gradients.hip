// The gated delta rule's gradients of q, k, the decays and beta, all chunks side by side, from the states before
// and the gradients of the states after each chunk.  Formulas and layouts: ftc_delta_kernel.h; with
//
//   P_ij = beta_j (dO_i . Z_j) D_ij rq_i rk_j  (j <= i),   R_ij = -beta_j (dE_i . Z_j) D_ij rk_i rk_j  (j < i)
//
//   dq_i = rq_i e^{G_i} S dO_i + sum_j P_ij k_j
//   dk+_i = -rk_i e^{G_i} S dE_i + sum_j R_ij k_j                  (k_i as it reads the state: with e^{+G_i})
//   dk-_j = rk_j beta_j e^{G_64 - G_j} dS Z_j + sum_i P_ij q_i + sum_i R_ij k_i      (as it is written: e^{-G_j})
//   dbeta_j = Z_j . dU_j - sum_{i > j} D_ij (k^_i . k^_j) (dE_i . Z_j)
//   dG_i = q_i . dq_i + k_i . dk+_i - k_i . dk-_i,  dG_64 += sum_j k_j . (first term of dk-_j) + e^{G_64} <S, dS>
//   dg_l = sum of dG_i over i >= l in the chunk
//   (normalised rows: dq - q (q . dq) / |q|^2, the same for k)
//
// A workgroup of four wavefronts takes a chunk of one key head and its value heads one after the other, so that the
// gradients of shared keys are summed in registers, in one order.  Phase 1 walks the columns of the state, 32 at a
// time through LDS; a wavefront has all 64 positions of a quarter of the key columns, and a quarter of the tiles of
// dO Z^T and dE Z^T.  Phase 2 multiplies the 64 x 64 matrices with the rows.
#include "ftc_delta_kernel.h"

namespace ftc {
namespace delta {
namespace {

constexpr int kThreads = 256;
constexpr int kSquare = Plane<128>::kBytes;  // a plane of 64 x 64

// A fragment-ordered block of 16 columns (TILES tiles of 16 rows) -> planes with a row per column
template <int TILES, int RB>
__device__ __forceinline__ void transpose_in(const float *from, lds_char *planes, int plane_bytes, int row0, int unit) {
    const int t = unit / 64, l = unit % 64;
    const f32x4 x = *(const f32x4a *)(from + 4 * unit);
    store_pieces(planes + Plane<RB>::addr(row0 + (l & 15), 4 * t + (l >> 4)), plane_bytes, x);
}

template <typename T, int KE>
__global__ __launch_bounds__(kThreads) void delta_gradients_kernel(DeltaArgs p) {
    constexpr int RB = 64 * KE, PIECES = Elem<T>::kPieces, ET = 2 * KE, EW = ET / 4;
    constexpr int kMB = 32;                                          // columns of the state at a time
    constexpr int kGo = kRows * 64, kSq = kMB * 128, kSt = kMB * RB;  // bytes of a plane of dO, of Z or dE, of a state
    constexpr int kPhase1 = PIECES * kGo + 6 * kSq + 6 * kSt;
    constexpr int kRowsPlane = Plane<RB>::kBytes;
    constexpr int kPhase2 = 2 * PIECES * kRowsPlane + 6 * kSquare;
    constexpr int kBytes = kPhase1 > kPhase2 ? kPhase1 : kPhase2;
    __shared__ __align__(16) char mem[kBytes];
    __shared__ __align__(16) float f_mem[kFactors * kRows];
    __shared__ float dots_mem[4][4][kRows];   // per wavefront: q.dq, k.dk+, k.dk-, k.(first term of dk-)
    __shared__ float total_mem[2][kRows];     // q.dq and k.dk of all value heads
    __shared__ float beta_mem[4][kRows];      // per row of tiles: the second term of dbeta
    __shared__ float state_mem[4];            // per wavefront: its share of <S, dS>
    lds_char *const lds = (lds_char *)mem;
    lds_char *const gop = lds, *const zp = gop + PIECES * kGo, *const dep = zp + 3 * kSq, *const sp = dep + 3 * kSq,
                    *const dsp = sp + 3 * kSt;
    lds_char *const qp = lds, *const kp = qp + PIECES * kRowsPlane, *const pp = kp + PIECES * kRowsPlane,
                    *const rp = pp + 3 * kSquare;
    lds_float *const fp = (lds_float *)f_mem;

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, q = lane >> 4;
    const int G = p.H / p.Hk;
    const int chunk = (int)(blockIdx.x % (uint32_t)p.chunks), nk = (int)(blockIdx.x / (uint32_t)p.chunks);
    const int n = nk / p.Hk, hk = nk % p.Hk;
    const int64_t l0 = (int64_t)chunk * kRows;
    const int rows = min((int64_t)kRows, p.L - l0);  // of the chunk in memory
    auto grad_at = [&](const Scalars &x, int h, int i) { return n * x.sn + h * x.sh + (l0 + i) * x.sl; };

    f32x4 dQ[4][EW] = {}, dK[4][EW] = {};
    if (tid < kRows) total_mem[0][tid] = total_mem[1][tid] = 0.f;

    for (int g = 0; g < G; g++) {
        const int h = hk * G + g;
        const Where w = where_of(p, n * p.H + h, chunk);
        if (w.valid == 0) {  // (the same for all heads of a sequence)
            if (tid < rows) {
                if (p.gg.ptr) store_from_f32(p.gg.ptr, p.gg.dtype, grad_at(p.gg, h, tid), 0.f);
                if (p.gb.ptr) store_from_f32(p.gb.ptr, p.gb.dtype, grad_at(p.gb, h, tid), 0.f);
            }
            continue;
        }
        const float *const factors = p.factors + w.at * (kFactors * kRows);
        for (int i = tid; i < kFactors * kRows; i += kThreads) fp[i] = factors[i];

        // ---- phase 1 ----
        f32x4 F[3] = {}, N[3] = {};                                   // (dO Z^T)^T, (dE Z^T)^T: rows j, columns i
        f32x4 aQ[4][EW] = {}, aP[4][EW] = {}, aM[4][EW] = {};         // S dO, S dE, dS Z
        float state_dot = 0.f;
        auto tile_of = [&](int x, int &ti, int &tj) {
            const int id = wave + 4 * x;
            ti = id < 2 ? 0 : id < 4 ? 1 : id < 8 ? 2 : 3, tj = id < 4 ? id & 1 : id & 3;
        };
        const __amdgpu_buffer_rsrc_t go_rows = chunk_rows(p.go, w.n, w.h, l0, Elem<T>::kBytes);
        for (int m0 = 0; m0 < p.col_blocks; m0 += 2) {
            RowTile<T, kMB, kThreads> go;
            // (32 columns from 16 m0 on: the offset goes into the rows' base)
            {
                Operand shifted = p.go;
                shifted.ptr = (const char *)p.go.ptr + (int64_t)m0 * kCols * Elem<T>::kBytes;
                const bool vec = (p.M - m0 * kCols) % (Elem<T>::kBytes == 4 ? 4 : 8) == 0 &&
                                 (((uintptr_t)shifted.ptr | (uint64_t)(shifted.stride_n * Elem<T>::kBytes) |
                                   (uint64_t)(shifted.stride_h * Elem<T>::kBytes) |
                                   (uint64_t)(shifted.stride_l * Elem<T>::kBytes)) & 15) == 0;
                go.load(chunk_rows(shifted, w.n, w.h, l0, Elem<T>::kBytes), (uint32_t)p.go.stride_l * Elem<T>::kBytes,
                        p.M - m0 * kCols, w.valid, vec, tid);
            }
            __syncthreads();  // (what was staged before has been read)
            go.template store<64>(gop, tid);
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const int block = m0 + b;
                const bool there = block < p.col_blocks;
                const int64_t at = w.at * p.col_blocks + (there ? block : m0);
                const float *const z = p.z + at * (4 * 256), *const de = p.de + at * (4 * 256),
                            *const s = p.s + at * (ET * 256), *const ds = p.ds + at * (ET * 256);
                if (there) {
                    transpose_in<4, 128>(z, zp, kSq, 16 * b, tid);
                    transpose_in<4, 128>(de, dep, kSq, 16 * b, tid);
#pragma unroll
                    for (int u = 0; u < ET / 4; u++) {
                        const int unit = tid + kThreads * u, t = unit / 64, l = unit % 64;
                        const f32x4 x = *(const f32x4a *)(s + 4 * unit), y = *(const f32x4a *)(ds + 4 * unit);
                        state_dot += (x[0] * y[0] + x[1] * y[1]) + (x[2] * y[2] + x[3] * y[3]);
                        store_pieces(sp + Plane<RB>::addr(16 * b + (l & 15), 4 * t + (l >> 4)), kSt, x);
                        store_pieces(dsp + Plane<RB>::addr(16 * b + (l & 15), 4 * t + (l >> 4)), kSt, y);
                    }
                } else {  // zeros: dO's columns past M are zero too
                    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                    const int t = tid / 64, l = tid % 64;
                    store_pieces(zp + Plane<128>::addr(16 * b + (l & 15), 4 * t + (l >> 4)), kSq, zero);
                    store_pieces(dep + Plane<128>::addr(16 * b + (l & 15), 4 * t + (l >> 4)), kSq, zero);
#pragma unroll
                    for (int u = 0; u < ET / 4; u++) {
                        const int unit = tid + kThreads * u, tt = unit / 64;
                        store_pieces(sp + Plane<RB>::addr(16 * b + (l & 15), 4 * tt + (l >> 4)), kSt, zero);
                        store_pieces(dsp + Plane<RB>::addr(16 * b + (l & 15), 4 * tt + (l >> 4)), kSt, zero);
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int x = 0; x < 3; x++) {
                int ti, tj;
                tile_of(x, ti, tj);
                Frag zf[3], of[PIECES], ef[3];
                columns_of<128>(zp, tj, 0, c, q, zf, kSq);
#pragma unroll
                for (int k = 0; k < PIECES; k++) of[k] = Plane<64>::rows(gop + k * kGo, ti, 0, c, q);
                F[x] = product(zf, of, F[x]);
                columns_of<128>(dep, ti, 0, c, q, ef, kSq);
                N[x] = product(zf, ef, N[x]);
            }
            Frag sf[EW][3], df[EW][3];
#pragma unroll
            for (int e = 0; e < EW; e++) {
                columns_of<RB>(sp, EW * wave + e, 0, c, q, sf[e], kSt);
                columns_of<RB>(dsp, EW * wave + e, 0, c, q, df[e], kSt);
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                Frag of[PIECES], ef[3], zf[3];
#pragma unroll
                for (int k = 0; k < PIECES; k++) of[k] = Plane<64>::rows(gop + k * kGo, t, 0, c, q);
                columns_of<128>(dep, t, 0, c, q, ef, kSq);
                columns_of<128>(zp, t, 0, c, q, zf, kSq);
#pragma unroll
                for (int e = 0; e < EW; e++) {
                    aQ[t][e] = product(of, sf[e], aQ[t][e]);
                    aP[t][e] = product(ef, sf[e], aP[t][e]);
                    aM[t][e] = product(zf, df[e], aM[t][e]);
                }
            }
        }
        (void)go_rows;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) state_dot += __shfl_xor(state_dot, d);
        if (lane == 0) state_mem[wave] = state_dot;

        // ---- phase 2 ----
        __syncthreads();
        {
            RowTile<T, 32 * KE, kThreads> tile;
            tile.load(chunk_rows(p.q, w.n, w.hk, l0, Elem<T>::kBytes), (uint32_t)p.q.stride_l * Elem<T>::kBytes, p.E,
                      w.valid, p.vec_q, tid);
            tile.template store<RB>(qp, tid);
            tile.load(chunk_rows(p.k, w.n, w.hk, l0, Elem<T>::kBytes), (uint32_t)p.k.stride_l * Elem<T>::kBytes, p.E,
                      w.valid, p.vec_k, tid);
            tile.template store<RB>(kp, tid);
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < 3; x++) {
            int ti, tj;
            tile_of(x, ti, tj);
            f32x4 kk = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KE; s++) {
                Frag a[PIECES], b[PIECES];
                rows_of<RB>(kp, tj, s, c, q, a);
                rows_of<RB>(kp, ti, s, c, q, b);
                kk = product(a, b, kk);
            }
            const int i = 16 * ti + c, j0 = 16 * tj + 4 * q;
            const float rk_i = fp[kRk * kRows + i], rq_i = fp[kRq * kRows + i];
            f32x4 pt, rt, bt;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int j = j0 + r;
                const float d = j <= i ? expf((fp[kHigh * kRows + i] - fp[kHigh * kRows + j]) +
                                              (fp[kLow * kRows + i] - fp[kLow * kRows + j])) * fp[kRk * kRows + j] : 0.f;
                const float b = fp[kBeta * kRows + j];
                pt[r] = j <= i ? b * F[x][r] * d * rq_i : 0.f;
                const float n_ij = j < i ? N[x][r] * d * rk_i : 0.f;
                rt[r] = -b * n_ij;
                bt[r] = sum16(n_ij * kk[r]);
            }
            store_pieces(pp + Plane<128>::addr(i, 4 * tj + q), kSquare, pt);
            store_pieces(rp + Plane<128>::addr(i, 4 * tj + q), kSquare, rt);
            if (c == 0)
#pragma unroll
                for (int r = 0; r < 4; r++) beta_mem[ti][j0 + r] = bt[r];
        }
        // the values of q and k at the places of the accumulators
        auto row_value = [&](const lds_char *planes, int row, int col) {
            float v = 0.f;
#pragma unroll
            for (int k = PIECES - 1; k >= 0; k--)
                v += bf16_to_f32(*(const __attribute__((address_space(3))) uint16_t *)(
                    planes + k * kRowsPlane + Plane<RB>::addr(row, col >> 2) + 2 * (col & 3)));
            return v;
        };
        float first[4][4];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * t + 4 * q + r;
                const float rise = fp[kRise * kRows + row], fall = fp[kFall * kRows + row], rk = fp[kRk * kRows + row];
                float dot = 0.f;
#pragma unroll
                for (int e = 0; e < EW; e++) {
                    aQ[t][e][r] *= rise * fp[kRq * kRows + row];
                    aP[t][e][r] *= -rise * rk;
                    aM[t][e][r] *= fall * rk * fp[kBeta * kRows + row];
                    dot = fmaf(row_value(kp, row, 16 * (EW * wave + e) + c), aM[t][e][r], dot);
                }
                first[t][r] = sum16(dot);
            }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag kf[EW][PIECES], qf[EW][PIECES];
#pragma unroll
            for (int e = 0; e < EW; e++) {
                columns_of<RB>(kp, EW * wave + e, s, c, q, kf[e]);
                columns_of<RB>(qp, EW * wave + e, s, c, q, qf[e]);
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                Frag f[3];
                if (t >= 2 * s) {  // rows i of tile t: columns j up to it
                    rows_of<128>(pp, t, s, c, q, f);
#pragma unroll
                    for (int e = 0; e < EW; e++) aQ[t][e] = product(f, kf[e], aQ[t][e]);
                    rows_of<128>(rp, t, s, c, q, f);
#pragma unroll
                    for (int e = 0; e < EW; e++) aP[t][e] = product(f, kf[e], aP[t][e]);
                }
                if (t < 2 * s + 2) {  // columns j of tile t: rows i from it on
                    columns_of<128>(pp, t, s, c, q, f);
#pragma unroll
                    for (int e = 0; e < EW; e++) aM[t][e] = product(f, qf[e], aM[t][e]);
                    columns_of<128>(rp, t, s, c, q, f);
#pragma unroll
                    for (int e = 0; e < EW; e++) aM[t][e] = product(f, kf[e], aM[t][e]);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * t + 4 * q + r;
                float dq = 0.f, dp = 0.f, dm = 0.f;
#pragma unroll
                for (int e = 0; e < EW; e++) {
                    const int col = 16 * (EW * wave + e) + c;
                    const float kv = row_value(kp, row, col);
                    dq = fmaf(row_value(qp, row, col), aQ[t][e][r], dq);
                    dp = fmaf(kv, aP[t][e][r], dp);
                    dm = fmaf(kv, aM[t][e][r], dm);
                }
                dq = sum16(dq), dp = sum16(dp), dm = sum16(dm);
                if (c == 0) {
                    dots_mem[wave][0][row] = dq, dots_mem[wave][1][row] = dp, dots_mem[wave][2][row] = dm;
                    dots_mem[wave][3][row] = first[t][r];
                }
#pragma unroll
                for (int e = 0; e < EW; e++) dQ[t][e][r] += aQ[t][e][r], dK[t][e][r] += aP[t][e][r] + aM[t][e][r];
            }
        __syncthreads();
        if (wave == 0) {
            float dot[4];
#pragma unroll
            for (int k = 0; k < 4; k++)
                dot[k] = (dots_mem[0][k][lane] + dots_mem[1][k][lane]) + (dots_mem[2][k][lane] + dots_mem[3][k][lane]);
            total_mem[0][lane] += dot[0], total_mem[1][lane] += dot[1] + dot[2];
            double sum = (double)dot[0] + (double)dot[1] - (double)dot[2], all = dot[3];
#pragma unroll
            for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d);
            all += (double)fp[kRise * kRows + kRows - 1] *
                   (((double)state_mem[0] + (double)state_mem[1]) + ((double)state_mem[2] + (double)state_mem[3]));
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {  // sums from here to the end
                const double other = __shfl_down(sum, d);
                if (lane + d < 64) sum += other;
            }
            if (p.gg.ptr && lane < rows)
                store_from_f32(p.gg.ptr, p.gg.dtype, grad_at(p.gg, h, lane), lane < w.valid ? (float)(sum + all) : 0.f);
        } else if (wave == 1 && p.gb.ptr && lane < rows) {
            float sum = 0.f;
            for (int b = 0; b < p.col_blocks; b++) sum += p.zdu[(w.at * p.col_blocks + b) * kRows + lane];
            // (tiles of column block lane / 16: rows of tiles from it on)
            float less = 0.f;
            for (int t = lane / 16; t < 4; t++) less += beta_mem[t][lane];
            store_from_f32(p.gb.ptr, p.gb.dtype, grad_at(p.gb, h, lane), lane < w.valid ? sum - less : 0.f);
        }
        __syncthreads();
    }

    const Where w = where_of(p, n * p.H + hk * G, chunk);
    if (w.valid > 0 && p.normalize) {  // (q, k, the factors of the last head: those of q and k are alike)
        auto row_value = [&](const lds_char *planes, int row, int col) {
            float v = 0.f;
#pragma unroll
            for (int k = PIECES - 1; k >= 0; k--)
                v += bf16_to_f32(*(const __attribute__((address_space(3))) uint16_t *)(
                    planes + k * kRowsPlane + Plane<RB>::addr(row, col >> 2) + 2 * (col & 3)));
            return v;
        };
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * t + 4 * q + r;
                const float rq = fp[kRq0 * kRows + row], rk = fp[kRk * kRows + row];
                const float fq = total_mem[0][row] * rq * rq, fk = total_mem[1][row] * rk * rk;
#pragma unroll
                for (int e = 0; e < EW; e++) {
                    const int col = 16 * (EW * wave + e) + c;
                    dQ[t][e][r] = fmaf(-fq, row_value(qp, row, col), dQ[t][e][r]);
                    dK[t][e][r] = fmaf(-fk, row_value(kp, row, col), dK[t][e][r]);
                }
            }
    }
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = 16 * t + 4 * q + r;
            if (row >= rows) continue;
#pragma unroll
            for (int e = 0; e < EW; e++) {
                const int col = 16 * (EW * wave + e) + c;
                if (col >= p.E) continue;
                if (p.gq.ptr)
                    store_from_f32(p.gq.ptr, p.gq.dtype,
                                   n * p.gq.stride_n + hk * p.gq.stride_h + (l0 + row) * p.gq.stride_l + col, dQ[t][e][r]);
                if (p.gk.ptr)
                    store_from_f32(p.gk.ptr, p.gk.dtype,
                                   n * p.gk.stride_n + hk * p.gk.stride_h + (l0 + row) * p.gk.stride_l + col, dK[t][e][r]);
            }
        }
}

template <typename T, int KE>
void launch(const DeltaArgs &p, hipStream_t stream) {
    const dim3 grid((uint32_t)p.N * (uint32_t)p.Hk * (uint32_t)p.chunks);
    delta_gradients_kernel<T, KE><<<grid, kThreads, 0, stream>>>(p);
}

}  // namespace

int delta_gradients(const DeltaArgs &p, bool bf16, hipStream_t stream) {
    if (p.E <= 64) bf16 ? launch<bf16_t, 2>(p, stream) : launch<float, 2>(p, stream);
    else bf16 ? launch<bf16_t, 4>(p, stream) : launch<float, 4>(p, stream);
    return FTC_OK;
}

}  // namespace delta
}  // namespace ftc
