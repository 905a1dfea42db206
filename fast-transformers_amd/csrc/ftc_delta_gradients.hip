// The gated delta rule's gradients of q, k, the decays and beta, all chunks side by side, from the states before
// and the gradients of the states after each chunk.  Formulas and layouts: ftc_delta_kernel.h; with
//
//   P_ij = beta_j (dO_i . Z_j) D_ij rq_i rk_j  (j <= i),   R_ij = -beta_j (dE_i . Z_j) D_ij rk_i rk_j  (j < i)
//
//   dq_i = rq_i e^{G_i} S dO_i + sum_j P_ij k_j
//   dk_i = -rk_i e^{G_i} S dE_i + sum_j R_ij k_j                               (k_i as it reads the state: e^{+G_i})
//          + rk_i beta_i e^{G_64 - G_i} dS Z_i + sum_j P_ji q_j + sum_j R_ji k_j           (as it is written: e^{-G_i})
//   (normalised rows: dq - q (q . dq) / |q|^2, the same for k)
//
// The other gradients need no more products than the reverse scan has made, since
//   q_i . dq_i = dO_i . O_i,   k_i . dk_i = -dE_i . (V_i - Z_i) as it reads and dE_i . Z_i as it is written:
//   dbeta_i = dE_i . Z_i / beta_i          (all terms of dE_i have the factor beta_i)
//   dG_i = dO_i . O_i - dE_i . V_i,   dg_l = sum of dG_i over i >= l in the chunk + <state after it, its gradient>
// (the last is e^{G_64} <S, dS> + what the chunk's keys write, taken anew in every chunk: nothing adds up over chunks).
//
// A workgroup of four or eight wavefronts takes a chunk of one key head and 64 of its columns, two to a compute unit, and the
// head's value heads one after the other, so that the gradients of shared keys are summed in registers, in one
// order.  Phase 1 walks the columns of the state, 32 at a time through LDS, the next 32 on their way meanwhile; a
// wavefront has 32 positions (of eight: 16) of 32 key columns, and its share of the tiles of dO Z^T and dE Z^T.  Phase 2 multiplies the
// 64 x 64 matrices with the rows.  What is not rows is in three pieces for bf16
// rows too: of a normalised row's gradient what lies along the row is taken away again, and may be nearly all of it.
//
// What bounds it: vector instructions, most of them cutting values into pieces (46 % of the time), LDS (35 %) and the matrix cores
// (25 %), two workgroups a compute unit, beside 2.2 GB of states, their gradients, Z, dE and rows.  Measured: 8192 chunks of
// 128 x 128 on 4096 of key heads, bf16, 860 to 910 us (2.5 TB/s; in two pieces 740 to 780); 1280 of 64 x 64, fp32, 94 to 97.
#include <type_traits>

#include "ftc_delta_kernel.h"

namespace ftc {
namespace delta {
namespace {

constexpr int kSlice = 64;  // key columns of a workgroup
// Wavefronts of a workgroup: four, two workgroups to a compute unit; rows in three pieces leave LDS for one workgroup, of eight.  (1280
// chunks of 64 x 64, fp32: 94 us, with four 111.  8192 of 128 x 128, bf16: 1224 with eight, with four 863.)
template <typename T>
constexpr int kWaves = Elem<T>::kPieces == 1 ? 4 : 8;

// The lane's column and row group anew: what is made of them belongs to the phase behind (all phases' addresses, held
// through the loop over heads, would not leave registers for the products)
__device__ __forceinline__ void renew(int &c, int &q) { asm volatile("" : "+v"(c), "+v"(q)); }
__device__ __forceinline__ int renewed(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

template <typename T>
__global__ __launch_bounds__(64 * kWaves<T>, 2) void delta_gradients_kernel(DeltaArgs p) {
    constexpr int PIECES = Elem<T>::kPieces, NP = 3;
    constexpr int RB = 2 * kSlice, EW = 2;
    constexpr int WAVES = kWaves<T>, kThreads = 64 * WAVES, RT = 8 / WAVES, XT = 12 / WAVES + (12 % WAVES != 0), BLOCKS = 8 / WAVES;
    constexpr int kMB = 32;                                // columns of the state at a time
    constexpr int kGo = kRows * 2 * kMB, kSq = kMB * 128;  // bytes of a plane of dO, of the others
    constexpr int kSquare = Plane<128>::kBytes;
    constexpr int kQK = 2 * PIECES * kSquare, kPhase1 = PIECES * kGo + 4 * NP * kSq, kPR = 2 * NP * kSquare;
    constexpr bool kResident = PIECES == 1;  // rows of q and k stay in LDS; else they come after phase 1
    constexpr int kBytes = kResident ? kQK + (kPhase1 > kPR ? kPhase1 : kPR) : (kPhase1 > kQK + kPR ? kPhase1 : kQK + kPR);
    __shared__ __align__(16) char mem[kBytes];
    __shared__ __align__(16) float f_mem[kFactors * kRows];
    __shared__ float dot_mem[2][WAVES / 4][kRows]; // of a value head: dE . Z, dE . V, by every other block of columns
    __shared__ float total_mem[2][kRows];  // q . dq and k . dk of all of them
    __shared__ float state_mem[WAVES];         // per wavefront: its share of <S, dS>
    lds_char *const lds = (lds_char *)mem;
    lds_char *const qp = lds, *const kp = qp + PIECES * kSquare;
    lds_char *const gop = lds + (kResident ? kQK : 0), *const zp = gop + PIECES * kGo, *const dep = zp + NP * kSq,
                    *const sp = dep + NP * kSq, *const dsp = sp + NP * kSq;
    lds_char *const pp = lds + kQK, *const rp = pp + NP * kSquare;
    lds_float *const fp = (lds_float *)f_mem;

    const int tid = threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6);
    int c = lane & 15, q = lane >> 4;
    const int e0 = EW * (wave & 1), t0 = RT * (wave >> 1);  // the wavefront's tiles of key columns and of positions
    // (workgroups go to the eight dies in turn: the slices of a chunk to the same)
    const int slices = (p.E + kSlice - 1) / kSlice, tiles = p.E <= 64 ? 4 : 8;
    const int turn = (int)(blockIdx.x >> 3), slice = scalar(turn % slices);
    const int unit_of = scalar((turn / slices) * 8 + (int)(blockIdx.x & 7));
    const int G = scalar(p.H / p.Hk);
    const int nk = scalar(unit_of / p.chunks), chunk = unit_of - nk * p.chunks;
    if (nk >= p.N * p.Hk) return;
    const int n = scalar(nk / p.Hk), hk = nk - n * p.Hk;
    const int64_t l0 = (int64_t)chunk * kRows;
    const int rows = (int)min((int64_t)kRows, p.L - l0);  // of the chunk in memory
    const int valid = where_of(p, n * p.H + hk * G, chunk).valid;  // (the same for all heads of a sequence)

    f32x4 dQ[RT][EW] = {}, dK[RT][EW] = {};
    auto slice_of = [&](const Operand &o) {
        Operand s = o;
        s.ptr = (const char *)o.ptr + slice * kSlice * Elem<T>::kBytes;
        return s;
    };
    auto stage_rows = [&]() {
        RowTile<T, kSlice, kThreads> tile;
        tile.load(chunk_rows(slice_of(p.q), n, hk, l0, Elem<T>::kBytes), (uint32_t)p.q.stride_l * Elem<T>::kBytes,
                  p.E - slice * kSlice, valid, p.vec_q, renewed(tid));
        tile.template store<RB>(qp, renewed(tid));
        tile.load(chunk_rows(slice_of(p.k), n, hk, l0, Elem<T>::kBytes), (uint32_t)p.k.stride_l * Elem<T>::kBytes,
                  p.E - slice * kSlice, valid, p.vec_k, renewed(tid));
        tile.template store<RB>(kp, renewed(tid));
    };

    // ---- what phase 1 stages of 32 columns: dO's rows (the first four wavefronts), and a tile of the fragments of either block ----
    RowTile<T, kMB, 256> go;
    const int tile = wave & 3, half = WAVES == 8 ? wave >> 2 : 0;  // (half: eight wavefronts have a block each)
    f32x4 zr[BLOCKS], er[BLOCKS], sr[BLOCKS], dr[BLOCKS];
    // (of v in its own type: widening it here would wait for it)
    using Raw = typename std::conditional<Elem<T>::kBytes == 4, uint32_t, uint16_t>::type;
    Raw vr[BLOCKS][4];
    auto request = [&](int h, int m0, bool any) {
        const int64_t at = ((int64_t)(n * p.H + h) * p.chunks + chunk) * p.col_blocks;
        const int l = renewed(lane);
        Operand shifted = p.go;
        shifted.ptr = (const char *)p.go.ptr + (int64_t)m0 * kCols * Elem<T>::kBytes;
        // (a block past the last one: zeros, from a buffer of no bytes or rows of no values)
        const int live = any ? valid : 0;
        if (wave < 4)
            go.load(chunk_rows(shifted, n, h, l0, Elem<T>::kBytes), (uint32_t)p.go.stride_l * Elem<T>::kBytes,
                    p.M - m0 * kCols, live, p.vec_go, 64 * wave + l);
        const __amdgpu_buffer_rsrc_t v_rows = chunk_rows(p.v, n, h, l0, Elem<T>::kBytes);
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
            const int block = m0 + half + b, col = block * kCols + (l & 15);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * tile + 4 * (l >> 4) + r;
                const bool in = (row < live) & (col < p.M);
                const uint32_t at = (uint32_t)row * ((uint32_t)p.v.stride_l * Elem<T>::kBytes) + (uint32_t)(col * Elem<T>::kBytes);
                const uint32_t from = in ? at : kOutside;
                if constexpr (Elem<T>::kBytes == 4) vr[b][r] = __builtin_amdgcn_raw_buffer_load_b32(v_rows, from, 0, 0);
                else vr[b][r] = __builtin_amdgcn_raw_buffer_load_b16(v_rows, from, 0, 0);
            }
            auto fragment = [&](const float *from, int count, int number) {
                const uint64_t base = (uint64_t)(from + ((at + block) * count + number) * 256);
                const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                    (void *)(((uint64_t)(uint32_t)scalar((int)(base >> 32)) << 32) | (uint32_t)scalar((int)(uint32_t)base)), 0,
                    any && block < p.col_blocks ? 1024 : 0, mfma::kRsrcFlags);
                return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, 16 * l, 0, 0));
            };
            zr[b] = fragment(p.z, 4, tile), er[b] = fragment(p.de, 4, tile);
            sr[b] = fragment(p.s, tiles, 4 * slice + tile), dr[b] = fragment(p.ds, tiles, 4 * slice + tile);
        }
    };
    // a fragment's place in planes with a row per column: four positions (or key columns) of column c
    auto put = [&](f32x4 &dot_z, f32x4 &dot_v) {
        const int l = renewed(lane), slot = 4 * tile + (l >> 4);
        if (wave < 4) go.template store<64>(gop, 64 * wave + l);
        float dot = 0.f;
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
            const int to = Plane<128>::addr(16 * (half + b) + (l & 15), slot);
            store_pieces(zp + to, kSq, zr[b]);
            store_pieces(dep + to, kSq, er[b]);
            store_pieces(sp + to, kSq, sr[b]);
            store_pieces(dsp + to, kSq, dr[b]);
            dot_z += er[b] * zr[b];
#pragma unroll
            for (int r = 0; r < 4; r++)
                dot_v[r] = fmaf(er[b][r], __uint_as_float(Elem<T>::kBytes == 4 ? (uint32_t)vr[b][r] : (uint32_t)vr[b][r] << 16), dot_v[r]);
            dot += (sr[b][0] * dr[b][0] + sr[b][1] * dr[b][1]) + (sr[b][2] * dr[b][2] + sr[b][3] * dr[b][3]);
        }
        return dot;
    };
    // the tiles of the square matrices, transposed: rows j of tile tj, columns i of tile ti
    auto tile_of = [&](int x, int &ti, int &tj) {
        const int id = min(wave + WAVES * x, 11);  // (twelve: four of eight wavefronts make the last one once more)
        ti = id < 2 ? 0 : id < 4 ? 1 : id < 8 ? 2 : 3, tj = id < 4 ? id & 1 : id & 3;
    };

    if (valid > 0) {
        request(hk * G, 0, true);
        if (kResident) stage_rows();
    }
    if (tid < kRows) total_mem[0][tid] = total_mem[1][tid] = 0.f;
    for (int g = 0; g < G && valid > 0; g++) {
        const int h = hk * G + g;
        const int64_t at = (int64_t)(n * p.H + h) * p.chunks + chunk;
        float o = 0.f;  // (dO . O of a row, for the normalisation)
        if (p.normalize && wave == 3)
            for (int b = 0; b < p.col_blocks; b++) o += p.dots[(at * p.col_blocks + b) * kRows + lane];
        static_assert(kFactors * kRows == 4 * 256, "four floats a lane");
        if (tid < 256)
            *(__attribute__((address_space(3))) f32x4a *)(fp + 4 * tid) = *(const f32x4a *)(p.factors + at * (kFactors * kRows) + 4 * tid);

        // ---- phase 1 ----
        f32x4 F[XT] = {}, N[XT] = {};                                    // (dO Z^T)^T, (dE Z^T)^T
        f32x4 aQ[RT][EW] = {}, aP[RT][EW] = {}, aM[RT][EW] = {};       // S dO, S dE, dS Z
        f32x4 dot_z = {0.f, 0.f, 0.f, 0.f}, dot_v = {0.f, 0.f, 0.f, 0.f};
        float state_dot = 0.f;
        for (int m0 = 0; m0 < p.col_blocks; m0 += 2) {
            __syncthreads();  // (what was staged before has been read)
            state_dot += put(dot_z, dot_v);
            __syncthreads();
            const bool more = m0 + 2 < p.col_blocks;
            request(more || g + 1 == G ? h : h + 1, more ? m0 + 2 : 0, more || g + 1 < G);
            renew(c, q);
#pragma unroll
            for (int x = 0; x < XT; x++) {
                int ti, tj;
                tile_of(x, ti, tj);
                Frag zf[NP], of[PIECES], ef[NP];
                columns_of<128>(zp, tj, 0, c, q, zf, kSq);
#pragma unroll
                for (int k = 0; k < PIECES; k++) of[k] = Plane<64>::rows(gop + k * kGo, ti, 0, c, q);
                F[x] = product(zf, of, F[x]);
                columns_of<128>(dep, ti, 0, c, q, ef, kSq);
                N[x] = product(zf, ef, N[x]);
            }
            Frag sf[EW][NP], df[EW][NP];
#pragma unroll
            for (int e = 0; e < EW; e++) {
                columns_of<RB>(sp, e0 + e, 0, c, q, sf[e], kSq);
                columns_of<RB>(dsp, e0 + e, 0, c, q, df[e], kSq);
            }
#pragma unroll
            for (int t = 0; t < RT; t++) {
                Frag of[PIECES], ef[NP], zf[NP];
#pragma unroll
                for (int k = 0; k < PIECES; k++) of[k] = Plane<64>::rows(gop + k * kGo, t0 + t, 0, c, q);
                columns_of<128>(dep, t0 + t, 0, c, q, ef, kSq);
                columns_of<128>(zp, t0 + t, 0, c, q, zf, kSq);
#pragma unroll
                for (int e = 0; e < EW; e++) {
                    aQ[t][e] = product(of, sf[e], aQ[t][e]);
                    aP[t][e] = product(ef, sf[e], aP[t][e]);
                    aM[t][e] = product(zf, df[e], aM[t][e]);
                }
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) state_dot += __shfl_xor(state_dot, d);
#pragma unroll
        for (int r = 0; r < 4; r++) dot_z[r] = sum16(dot_z[r]), dot_v[r] = sum16(dot_v[r]);
        settle();
        if (lane == 0) state_mem[wave] = state_dot;
        if (c == 0)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                dot_mem[0][half][16 * tile + 4 * q + r] = dot_z[r];
                dot_mem[1][half][16 * tile + 4 * q + r] = dot_v[r];
            }

        // ---- phase 2 ----
        __syncthreads();
        renew(c, q);
        if (!kResident) stage_rows();
#pragma unroll
        for (int x = 0; x < XT; x++) {
            int ti, tj;
            tile_of(x, ti, tj);
            const int i = 16 * ti + c, j0 = 16 * tj + 4 * q;
            const float rk_i = fp[kRkBack * kRows + i], rq_i = fp[kRq * kRows + i];
            f32x4 pt, rt;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int j = j0 + r;
                const float d = j <= i ? expf((fp[kHigh * kRows + i] - fp[kHigh * kRows + j]) +
                                              (fp[kLow * kRows + i] - fp[kLow * kRows + j])) *
                                             (fp[kRk * kRows + j] * fp[kBeta * kRows + j]) : 0.f;
                pt[r] = j <= i ? F[x][r] * d * rq_i : 0.f;
                rt[r] = j < i ? -N[x][r] * d * rk_i : 0.f;
            }
            store_pieces(pp + Plane<128>::addr(i, 4 * tj + q), kSquare, pt);
            store_pieces(rp + Plane<128>::addr(i, 4 * tj + q), kSquare, rt);
        }
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * (t0 + t) + 4 * q + r;
                const float read_q = fp[kReadQ * kRows + row], read_k = fp[kReadBack * kRows + row], write = fp[kWrite * kRows + row];
#pragma unroll
                for (int e = 0; e < EW; e++) {
                    dQ[t][e][r] = fmaf(read_q, aQ[t][e][r], dQ[t][e][r]);
                    dK[t][e][r] += write * aM[t][e][r] - read_k * aP[t][e][r];
                }
            }
        // what the decays' and beta's gradients are made of, for the kernel behind
        auto dots_of = [&](int which) {
            return WAVES == 8 ? dot_mem[which][0][lane] + dot_mem[which][WAVES / 4 - 1][lane] : dot_mem[which][0][lane];
        };
        if (wave < 2) {
            if (slice == 0) p.sums[at * kSums + kRows * wave + lane] = dots_of(wave);
        } else if (wave == 2) {
            float state = (state_mem[0] + state_mem[1]) + (state_mem[2] + state_mem[3]);
            if (WAVES == 8)
                state += (state_mem[WAVES - 4] + state_mem[WAVES - 3]) + (state_mem[WAVES - 2] + state_mem[WAVES - 1]);
            if (lane == 0) p.sums[at * kSums + 2 * kRows + slice] = state;
        } else if (p.normalize && wave == 3) {
            total_mem[0][lane] += o, total_mem[1][lane] += fp[kRkBack * kRows + lane] == 0.f ? 0.f : 2.f * dots_of(0) - dots_of(1);
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag kf[EW][PIECES], qf[EW][PIECES];
#pragma unroll
            for (int e = 0; e < EW; e++) {
                columns_of<RB>(kp, e0 + e, s, c, q, kf[e]);
                columns_of<RB>(qp, e0 + e, s, c, q, qf[e]);
            }
#pragma unroll
            for (int t = 0; t < RT; t++) {
                Frag f[NP];
                if (t0 + t >= 2 * s) {  // rows i: columns j up to it
                    rows_of<128>(pp, t0 + t, s, c, q, f);
#pragma unroll
                    for (int e = 0; e < EW; e++) dQ[t][e] = product(f, kf[e], dQ[t][e]);
                    rows_of<128>(rp, t0 + t, s, c, q, f);
#pragma unroll
                    for (int e = 0; e < EW; e++) dK[t][e] = product(f, kf[e], dK[t][e]);
                }
                if (t0 + t < 2 * s + 2) {  // columns j: rows i from it on
                    columns_of<128>(pp, t0 + t, s, c, q, f);
#pragma unroll
                    for (int e = 0; e < EW; e++) dK[t][e] = product(f, qf[e], dK[t][e]);
                    columns_of<128>(rp, t0 + t, s, c, q, f);
#pragma unroll
                    for (int e = 0; e < EW; e++) dK[t][e] = product(f, kf[e], dK[t][e]);
                }
            }
        }
        settle();
        __syncthreads();
    }

    renew(c, q);
    if (valid > 0 && p.normalize) {  // (the factors of the last head: those of q and k are alike)
        const bool one = p.E == 1;
        auto row_value = [&](const lds_char *planes, int row, int col) {
            float v = 0.f;
#pragma unroll
            for (int k = PIECES - 1; k >= 0; k--)
                v += bf16_to_f32(*(const __attribute__((address_space(3))) uint16_t *)(
                    planes + k * kSquare + Plane<RB>::addr(row, col >> 2) + 2 * (col & 3)));
            return v;
        };
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * (t0 + t) + 4 * q + r;
                const float rq = fp[kRq0 * kRows + row], rk = fp[kRk * kRows + row];
                // (of a row of one value eps / (x^2 + eps) is left, which the difference would lose)
                const float fq = one ? 0.f : total_mem[0][row] * rq * rq, fk = one ? 0.f : total_mem[1][row] * rk * rk;
                const float left_q = one ? kNormEps * rq * rq : 1.f, left_k = one ? kNormEps * rk * rk : 1.f;
#pragma unroll
                for (int e = 0; e < EW; e++) {
                    const int col = 16 * (e0 + e) + c;
                    dQ[t][e][r] = fmaf(-fq, row_value(qp, row, col), left_q * dQ[t][e][r]);
                    dK[t][e][r] = fmaf(-fk, row_value(kp, row, col), left_k * dK[t][e][r]);
                }
            }
    }
    // (a buffer drops what lies outside)
    auto leave = [&](const OperandOut &out, const f32x4 (&x)[RT][EW]) {
        if (!out.ptr) return;
        const __amdgpu_buffer_rsrc_t rs = chunk_rows(Operand{out.ptr, out.stride_n, out.stride_h, out.stride_l, 0, 0}, n, hk, l0,
                                                     Elem<T>::kBytes);
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int e = 0; e < EW; e++) {
                    const int row = 16 * (t0 + t) + 4 * q + r, col = slice * kSlice + 16 * (e0 + e) + c;
                    const uint32_t to = row < rows && col < p.E
                        ? (uint32_t)row * ((uint32_t)out.stride_l * Elem<T>::kBytes) + (uint32_t)(col * Elem<T>::kBytes) : kOutside;
                    if (Elem<T>::kBytes == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[t][e][r]), rs, to, 0, 0);
                    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (__bf16)x[t][e][r]), rs, to, 0, 0);
                }
    };
    leave(p.gq, dQ);
    leave(p.gk, dK);
}

// The gradients of the decays and of beta: a workgroup per chunk and chain, a lane per position.
//
// The sums of dG take back what each pair of positions added to it except where the pair lies astride l; what is left over of the
// rest is rounding, 2^-22 or so of a position's dO . O.  That is nothing beside what lies astride, unless there are only
// a few positions or all decays are strong.  Such chunks add up what lies astride itself: pairs up to kBand positions
// apart, reads of the state by the first 16 positions and writes to it by the last; what is further off has faded
// by e^{kStrong (kBand + 1)} = 2^-28.  Products on the fp32 matrix instruction, whose operands are values as they are.
constexpr int kFew = 4;            // positions
constexpr int kBand = 9;
constexpr float kStrong = -2.f;    // the weakest log decay (the rounding is then below 2^-19 of what lies astride)
constexpr int kPairs = kRows * 33;  // pairs (i, j) in LDS, at 33 i + j - 16 (i / 16) + 16
constexpr int kAstride = kPairs + 4 * (16 + kRows);  // ... and each wavefront's sums of reads and of writes

// By the four wavefronts of a workgroup: 16 positions' pairs each, and every fourth block of columns.  Measured (E = M = 128, bf16): a
// chunk of 1 to 4 positions 26 us, of 64 strong ones 27, 8192 of them 650 (of others the whole kernel takes 4, 4 and 26).
// VEC: rows can be read 16 bytes at a time (here 8, or 16).
template <typename T, bool VEC>
__device__ __forceinline__ void find_astride(const DeltaArgs &p, const Where &w, int wave, int lane, lds_float *mem) {
    constexpr uint32_t B = Elem<T>::kBytes;
    const int c = lane & 15, q4 = lane / 16 * 4, valid = scalar(w.valid), tiles = p.E <= 64 ? 4 : 8;
    const int64_t l0 = (int64_t)w.chunk * kRows;
    const float *const factors = p.factors + w.at * (kFactors * kRows);
    const float *const Z = p.z + w.at * p.col_blocks * 1024, *const dE = p.de + w.at * p.col_blocks * 1024;
    const auto rq = chunk_rows(p.q, w.n, w.hk, l0, B), rk = chunk_rows(p.k, w.n, w.hk, l0, B), ro = chunk_rows(p.go, w.n, w.h, l0, B);
    const uint32_t sq = (uint32_t)p.q.stride_l * B, sk = (uint32_t)p.k.stride_l * B, so = (uint32_t)p.go.stride_l * B;
    // four values of a row from column `col`; four rows' values of one column; a result's tile with its rows in the lanes
    auto along = [&](__amdgpu_buffer_rsrc_t rs, uint32_t stride, int width, int row, int col) {
        f32x4 x;
        if (VEC) {
            const uint32_t at = row < valid && col < width ? (uint32_t)row * stride + (uint32_t)col * B : kOutside;
            if (B == 4) return __builtin_bit_cast(f32x4, (u32x4)__builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0));
            const u32x2 two = __builtin_amdgcn_raw_buffer_load_b64(rs, at, 0, 0);
            return f32x4{__uint_as_float(two.x << 16), __uint_as_float(two.x & 0xffff0000u), __uint_as_float(two.y << 16),
                         __uint_as_float(two.y & 0xffff0000u)};
        }
#pragma unroll
        for (int r = 0; r < 4; r++)
            x[r] = load_one<T>(rs, row < valid && col + r < width ? (uint32_t)row * stride + (uint32_t)(col + r) * B : kOutside);
        return x;
    };
    auto down = [&](int row, int col) {
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; r++)
            x[r] = load_one<T>(ro, row + r < valid && col < p.M ? (uint32_t)(row + r) * so + (uint32_t)col * B : kOutside);
        return x;
    };
    auto turned = [&](const float *of, int b, int t) {  // row 16 t + c, columns 16 b + q4 ..
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; r++) x[r] = of[b * 1024 + t * 256 + c / 4 * 64 + (q4 + r) * 4 + c % 4];
        return x;
    };
    lds_float *const pairs = mem, *const reads = mem + kPairs + wave * (16 + kRows), *const writes = reads + 16;

    if (16 * wave < valid) {
        const int ti = wave;
        f32x4 P[2] = {}, R[2] = {}, A[2] = {}, K[2] = {};  // pairs of a position with those of its tile and of the tile before
        const int before = ti > 0 ? ti - 1 : 0;
#pragma unroll 4
        for (int b = 0; b < p.col_blocks; b++) {
            const f32x4 o = along(ro, so, p.M, 16 * ti + c, 16 * b + q4), e = turned(dE, b, ti);
            const f32x4 z0 = turned(Z, b, ti), z1 = turned(Z, b, before);
            P[0] = mfma4(o, z0, P[0]), R[0] = mfma4(e, z0, R[0]), P[1] = mfma4(o, z1, P[1]), R[1] = mfma4(e, z1, R[1]);
        }
#pragma unroll 4
        for (int t = 0; t < tiles; t++) {
            const f32x4 q = along(rq, sq, p.E, 16 * ti + c, 16 * t + q4), k0 = along(rk, sk, p.E, 16 * ti + c, 16 * t + q4);
            const f32x4 k1 = along(rk, sk, p.E, 16 * before + c, 16 * t + q4);
            A[0] = mfma4(q, k0, A[0]), K[0] = mfma4(k0, k0, K[0]), A[1] = mfma4(q, k1, A[1]), K[1] = mfma4(k0, k1, K[1]);
        }
        settle();
#pragma unroll
        for (int back = 0; back < 2; back++) {
            const int j = 16 * (ti - back) + c, from = j < 0 ? 0 : j;
            const float beta = factors[kBeta * kRows + from] * factors[kRk * kRows + from];
            const float high = factors[kHigh * kRows + from], low = factors[kLow * kRows + from];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = 16 * ti + q4 + r;
                const float fade = expf((factors[kHigh * kRows + i] - high) + (factors[kLow * kRows + i] - low));
                const float x = factors[kRq * kRows + i] * A[back][r] * P[back][r] - factors[kRkBack * kRows + i] * K[back][r] * R[back][r];
                pairs[33 * i + c + 16 - 16 * back] = j >= 0 && j < i && i < valid ? fade * beta * x : 0.f;
            }
        }
    }
    // what positions 0 to 15 read of the state before the chunk, and what the last ones' two tiles write to the one after
    const int last = (valid - 1) / 16, but_one = last > 0 ? last - 1 : 0;
    const f32x4 by_q = *(const f32x4a *)(factors + kReadQ * kRows + q4), by_k = *(const f32x4a *)(factors + kReadBack * kRows + q4);
    const f32x4 by0 = *(const f32x4a *)(factors + kWrite * kRows + 16 * last + q4);
    const f32x4 by1 = *(const f32x4a *)(factors + kWrite * kRows + 16 * but_one + q4);
    f32x4 read = {0.f, 0.f, 0.f, 0.f}, write0 = read, write1 = read;
    for (int b = wave; b < p.col_blocks; b += 4) {
        const float *const S = p.s + ((w.at * p.col_blocks + b) * tiles * 64 + lane) * 4;
        const float *const dS = p.ds + ((w.at * p.col_blocks + b) * tiles * 64 + lane) * 4;
        const f32x4 o = down(q4, 16 * b + c), e = *(const f32x4a *)(dE + b * 1024 + lane * 4);
        const f32x4 z0 = *(const f32x4a *)(Z + b * 1024 + last * 256 + lane * 4);
        const f32x4 z1 = *(const f32x4a *)(Z + b * 1024 + but_one * 256 + lane * 4);
        f32x4 yq = {0.f, 0.f, 0.f, 0.f}, yk = yq, y0 = yq, y1 = yq;
#pragma unroll 4
        for (int t = 0; t < tiles; t++) {
            const f32x4 s = *(const f32x4a *)(S + 256 * t), ds = *(const f32x4a *)(dS + 256 * t);
            const f32x4 q = along(rq, sq, p.E, c, 16 * t + q4), k = along(rk, sk, p.E, c, 16 * t + q4);
            const f32x4 k0 = along(rk, sk, p.E, 16 * last + c, 16 * t + q4), k1 = along(rk, sk, p.E, 16 * but_one + c, 16 * t + q4);
            yq = mfma4(q, s, yq), yk = mfma4(k, s, yk), y0 = mfma4(k0, ds, y0), y1 = mfma4(k1, ds, y1);
        }
        settle();
        read += by_q * yq * o - by_k * yk * e, write0 += by0 * y0 * z0, write1 += by1 * y1 * z1;
    }
    auto leave = [&](lds_float *to, int row, const f32x4 &sum) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            float x = row + r < valid ? sum[r] : 0.f;
#pragma unroll
            for (int d = 1; d < 16; d *= 2) x += __shfl_xor(x, d);
            if (c == 0) to[row + r] = x;
        }
    };
    writes[lane] = 0.f;
    leave(reads, q4, read);
    if (last > 0) leave(writes, 16 * but_one + q4, write1);
    leave(writes, 16 * last + q4, write0);
}
// the lane's position of what find_astride left
__device__ __forceinline__ float add_astride(const lds_float *mem, int valid, int lane) {
    const lds_float *const reads = mem + kPairs, *const writes = reads + 16;
    constexpr int kNext = 16 + kRows;
    float dg = 0.f, wrote = writes[lane] + writes[kNext + lane] + writes[2 * kNext + lane] + writes[3 * kNext + lane];
    float read = lane < 16 ? reads[lane] + reads[kNext + lane] + reads[2 * kNext + lane] + reads[3 * kNext + lane] : 0.f;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {  // (reads from here on, writes up to here)
        const float later = __shfl_down(read, d), earlier = __shfl_up(wrote, d);
        if (lane + d < 64) read += later;
        if (lane >= d) wrote += earlier;
    }
    wrote = __shfl_up(wrote, 1);
    dg = read + (lane > 0 ? wrote : 0.f);
#pragma unroll
    for (int s = kBand - 1; s >= 0; s--) {
        const int i = lane + s, at = 33 * i - i / 16 * 16 + 16;
#pragma unroll
        for (int back = s + 1; back <= kBand; back++)
            if (i < valid && i >= back) dg += mem[at + i - back];
    }
    return dg;
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256, 4) void delta_decays_kernel(DeltaArgs p) {
    __shared__ float astride_mem[kAstride], sums_mem[2][4][kRows];
    const int tid = threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6);
    const int chain = scalar((int)(blockIdx.x / (uint32_t)p.chunks));
    const Where w = where_of(p, chain, (int)(blockIdx.x - (uint32_t)chain * (uint32_t)p.chunks));
    float dg = 0.f, db = 0.f;
    if (w.valid > 0) {
        const float *const sums = p.sums + w.at * kSums, *const factors = p.factors + w.at * (kFactors * kRows);
        float o = 0.f, written = 0.f;
#pragma unroll 2
        for (int b = wave; b < p.col_blocks; b += 4) {
            o += p.dots[(w.at * p.col_blocks + b) * kRows + lane];
            written += p.written[(w.at * p.col_blocks + b) * 64 + lane];
        }
        const float z = sums[lane], v = sums[kRows + lane], beta = factors[kBetaBack * kRows + lane];
        const float high = factors[kHigh * kRows + lane], before = __shfl_up(high, 1);
        const bool apart = w.valid <= kFew || __all(lane == 0 || lane >= w.valid || high - before <= kStrong);
        sums_mem[0][wave][lane] = o, sums_mem[1][wave][lane] = written;
        if (apart) find_astride<T, VEC>(p, w, wave, lane, (lds_float *)astride_mem);
        __syncthreads();
        if (wave > 0) return;
        const float state = p.E <= kSlice ? sums[2 * kRows] : sums[2 * kRows] + sums[2 * kRows + 1];
        const float through = factors[kRise * kRows + kRows - 1] * state;
        if (apart) {
            dg = through + add_astride((const lds_float *)astride_mem, w.valid, lane);
        } else {
            auto all_of = [&](int i) { return (sums_mem[i][0][lane] + sums_mem[i][1][lane]) + (sums_mem[i][2][lane] + sums_mem[i][3][lane]); };
            // (a beta that the backward has for zero: neither read nor written)
            const bool shut = beta == kLeastBeta;
            double sum = (double)all_of(0) - (double)(shut ? 0.f : v), all = __all(shut || lane >= w.valid) ? 0.f : all_of(1);
#pragma unroll
            for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d);
            all += (double)through;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {  // sums from here to the end
                const double other = __shfl_down(sum, d);
                if (lane + d < 64) sum += other;
            }
            dg = (float)(sum + all);
        }
        db = z / beta;
    }
    const int64_t l = (int64_t)w.chunk * kRows + lane;
    if (wave > 0 || l >= p.L) return;
    if (lane >= w.valid) dg = db = 0.f;
    if (p.gg.ptr) store_from_f32(p.gg.ptr, p.gg.dtype, w.n * p.gg.sn + w.h * p.gg.sh + l * p.gg.sl, dg);
    if (p.gb.ptr) store_from_f32(p.gb.ptr, p.gb.dtype, w.n * p.gb.sn + w.h * p.gb.sh + l * p.gb.sl, db);
}

}  // namespace

int delta_gradients(const DeltaArgs &p, bool bf16, hipStream_t stream) {
    const uint32_t slices = (uint32_t)((p.E + kSlice - 1) / kSlice);
    const dim3 grid(((uint32_t)p.N * (uint32_t)p.Hk * (uint32_t)p.chunks + 7) / 8 * 8 * slices);
    if (bf16) delta_gradients_kernel<bf16_t><<<grid, 64 * kWaves<bf16_t>, 0, stream>>>(p);
    else delta_gradients_kernel<float><<<grid, 64 * kWaves<float>, 0, stream>>>(p);
    if (p.gg.ptr || p.gb.ptr) {
        const dim3 units((uint32_t)p.N * (uint32_t)p.H * (uint32_t)p.chunks);
        const bool vec = p.vec_q && p.vec_k && p.vec_go;
        (bf16 ? vec ? delta_decays_kernel<bf16_t, true> : delta_decays_kernel<bf16_t, false>
              : vec ? delta_decays_kernel<float, true> : delta_decays_kernel<float, false>)<<<units, 256, 0, stream>>>(p);
    }
    return FTC_OK;
}

}  // namespace delta
}  // namespace ftc
