// The gated delta rule's state from chunk to chunk, forward (Z of every position, the state before every chunk and
// after the last) and backward (the gradient of the state, dE = dV).  Formulas and layouts: ftc_delta_kernel.h.
//
// A wavefront owns 16 columns of one chain's state in registers and walks the chunks, alone: what it multiplies with
// it reads as fragments, straight into the registers of the operands, each one's next chunk requested as soon as this
// chunk's is used.  A chunk is a chain of dependent products, so what bounds few chains is its latency.
#include "ftc_delta_kernel.h"

namespace ftc {
namespace delta {
namespace {

// Keeps the requests of a phase where they are written
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

// rows 16 t + 4 q .. of a factor
__device__ __forceinline__ void load_factor(const float *f, int which, int q, f32x4 (&x)[4]) {
#pragma unroll
    for (int t = 0; t < 4; t++) x[t] = *(const f32x4a *)(f + which * kRows + 16 * t + 4 * q);
}
__device__ __forceinline__ void load_tiles(const float *from, f32x4 (&x)[4]) {
#pragma unroll
    for (int t = 0; t < 4; t++) x[t] = *(const f32x4a *)(from + 256 * t);
}
__device__ __forceinline__ void store_tiles(float *to, const f32x4 (&x)[4]) {
#pragma unroll
    for (int t = 0; t < 4; t++) *(f32x4a *)(to + 256 * t) = x[t];
}

// acc += A B with the left operand's fragment held, or read here
template <bool HELD, int HA, int NB>
__device__ __forceinline__ f32x4 times(const Frag (&held)[HA], const uint16_t *from, int number, int lane, const Frag (&b)[NB],
                                       f32x4 acc) {
    if constexpr (HELD) {
        return product(held, b, acc);
    } else {
        Frag a[3];
        load_frag(from, number, lane, a);
        return product(a, b, acc);
    }
}

// Workgroups go to the eight dies in turn: those of one chain to the same, whose cache they share
__device__ __forceinline__ bool place(const DeltaArgs &p, int groups, int &chain, int &group) {
    const uint32_t die = blockIdx.x % 8u, slot = blockIdx.x / 8u;
    chain = (int)(slot / (uint32_t)groups * 8u + die), group = (int)(slot % (uint32_t)groups);
    return chain < p.N * p.H;
}

// Values of rows 16 t + 4 q + r of a column, as they come from memory: what is done to them here would wait for them
template <typename T>
struct Column {
    uint32_t raw[4][4];
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t row_bytes, int col, int width, int valid, int q) {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * t + 4 * q + r;
                const uint32_t at = row < valid && col < width
                                        ? (uint32_t)row * row_bytes + (uint32_t)(col * Elem<T>::kBytes) : kOutside;
                raw[t][r] = Elem<T>::kBytes == 4 ? __builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, 0)
                                                 : (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(rs, at, 0, 0);
            }
    }
    __device__ __forceinline__ f32x4 values(int t) const {
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; r++) x[r] = __uint_as_float(Elem<T>::kBytes == 4 ? raw[t][r] : raw[t][r] << 16);
        return x;
    }
};

template <typename T, int KE, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(1, 1))) void delta_scan_kernel(DeltaArgs p) {
    constexpr int PIECES = Elem<T>::kPieces, ET = 2 * KE, kKeys = 4 * KE * PIECES * 512;
    const int lane = threadIdx.x & 63, wave = scalar(threadIdx.x >> 6), c = lane & 15, q = lane >> 4;
    int chain, group;
    if (!place(p, (p.col_blocks + NW - 1) / NW, chain, group)) return;
    const int block = group * NW + wave, col = kCols * block + c;
    if (block >= p.col_blocks) return;
    const Where w = where_of(p, chain, 0);
    const int chunks = chunks_of(w.len);

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

    const uint32_t v_row = (uint32_t)p.v.stride_l * Elem<T>::kBytes;
    // (three pieces of wide rows would not fit: read when they are used)
    constexpr bool kHold = KE * PIECES <= 6;
    Frag kr[4 * KE][kHold ? PIECES : 1], kc[4 * KE][kHold ? PIECES : 1], tf[kTFrags][3];
    Column<T> V;
    f32x4 in[4], out[4];
    float last;
    auto load_in = [&](int chunk) {
        if constexpr (kHold)
#pragma unroll
            for (int i = 0; i < 4 * KE; i++) load_frag(p.kr + (w.key_at + chunk) * kKeys, i, lane, kr[i]);
    };
    auto load_values = [&](int chunk) {
        V.load(chunk_rows(p.v, w.n, w.h, (int64_t)chunk * kRows, Elem<T>::kBytes), v_row, col, p.M,
               min(kRows, w.len - chunk * kRows), q);
        load_factor(p.factors + (w.at + chunk) * (kFactors * kRows), kReadK, q, in);
    };
    auto load_t = [&](int chunk) {
#pragma unroll
        for (int i = 0; i < kTFrags; i++) load_frag(p.t + (w.at + chunk) * (kTFrags * 3 * 512), i, lane, tf[i]);
        load_factor(p.factors + (w.at + chunk) * (kFactors * kRows), kWrite, q, out);
        last = p.factors[(w.at + chunk) * (kFactors * kRows) + kRise * kRows + kRows - 1];
    };
    auto load_out = [&](int chunk) {
        if constexpr (kHold)
#pragma unroll
            for (int i = 0; i < 4 * KE; i++) load_frag(p.kc + (w.key_at + chunk) * kKeys, i, lane, kc[i]);
    };
    if (chunks > 0) load_in(0), load_values(0), load_t(0), load_out(0);
    for (int chunk = 0; chunk < chunks; chunk++) {
        const int64_t at = (w.at + chunk) * p.col_blocks + block;
        const int next = min(chunk + 1, chunks - 1);
        {
            float *const to = p.s + at * (ET * 256) + 4 * lane;
#pragma unroll
            for (int t = 0; t < ET; t++) *(f32x4a *)(to + 256 * t) = S[t];
        }
        // E = V - diag(rk e^G) K S
        f32x4 P[4] = {}, Z[4] = {};
#pragma unroll
        for (int s = 0; s < KE; s++) {
            Frag sf[3];
            cut(S[2 * s], S[2 * s + 1], sf);
#pragma unroll
            for (int t = 0; t < 4; t++) P[t] = times<kHold>(kr[t * KE + s], p.kr + (w.key_at + chunk) * kKeys, t * KE + s, lane, sf, P[t]);
        }
#pragma unroll
        for (int t = 0; t < 4; t++) P[t] = V.values(t) - in[t] * P[t];
        phase();
        load_in(next), load_values(next);
        phase();
        // Z = T E (tiles above the diagonal are zero)
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag ef[3];
            cut(P[2 * s], P[2 * s + 1], ef);
#pragma unroll
            for (int t = 2 * s; t < 4; t++) Z[t] = product(tf[t_number(t, s)], ef, Z[t]);
        }
        store_tiles(p.z + at * (4 * 256) + 4 * lane, Z);
        // S <- e^{G_64} S + K^T diag(rk beta e^{G_64 - G}) Z
#pragma unroll
        for (int t = 0; t < 4; t++) Z[t] *= out[t];
#pragma unroll
        for (int t = 0; t < ET; t++) S[t] *= last;
        phase();
        load_t(next);
        phase();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag uf[3];
            cut(Z[2 * s], Z[2 * s + 1], uf);
#pragma unroll
            for (int t = 0; t < ET; t++)
                S[t] = times<kHold>(kc[2 * t + s], p.kc + (w.key_at + chunk) * kKeys, 2 * t + s, lane, uf, S[t]);
        }
        phase();
        load_out(next);
        phase();
    }
    if (p.final_.ptr)
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
// and what the chunk's keys write of <state, its gradient>: the sum of beta Z . diag(rk e^{G_64 - G}) K dS.
template <typename T, int KE, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(1, 1))) void delta_scan_back_kernel(DeltaArgs p) {
    constexpr int PIECES = Elem<T>::kPieces, ET = 2 * KE, kKeys = 4 * KE * PIECES * 512;
    const int lane = threadIdx.x & 63, wave = scalar(threadIdx.x >> 6), c = lane & 15, q = lane >> 4;
    int chain, group;
    if (!place(p, (p.col_blocks + NW - 1) / NW, chain, group)) return;
    const int block = group * NW + wave, col = kCols * block + c;
    if (block >= p.col_blocks) return;
    const Where w = where_of(p, chain, 0);
    const int chunks = chunks_of(w.len);

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

    const uint32_t g_row = (uint32_t)p.go.stride_l * Elem<T>::kBytes, gv_row = (uint32_t)p.gv.stride_l * Elem<T>::kBytes;
    constexpr bool kHold = KE * PIECES <= 4;
    Frag kr[4 * KE][kHold ? PIECES : 1], kc[4 * KE][kHold ? PIECES : 1], qc[4 * KE][kHold ? PIECES : 1], tf[kTFrags][3];
    Column<T> Gr;
    f32x4 Y[4], Z[4], write[4], beta[4], read_q[4], read_k[4];
    float last;
    auto factors = [&](int chunk) { return p.factors + (w.at + chunk) * (kFactors * kRows); };
    auto tiles = [&](int chunk) { return ((w.at + chunk) * p.col_blocks + block) * (4 * 256) + 4 * lane; };
    auto load_in = [&](int chunk) {
        if constexpr (kHold)
#pragma unroll
            for (int i = 0; i < 4 * KE; i++) load_frag(p.kr + (w.key_at + chunk) * kKeys, i, lane, kr[i]);
        load_factor(factors(chunk), kWrite, q, write);
        load_factor(factors(chunk), kBeta, q, beta);
        load_tiles(p.de + tiles(chunk), Y);
        load_tiles(p.z + tiles(chunk), Z);
    };
    auto load_t = [&](int chunk) {
#pragma unroll
        for (int i = 0; i < kTFrags; i++) load_frag(p.tt + (w.at + chunk) * (kTFrags * 3 * 512), i, lane, tf[i]);
        load_factor(factors(chunk), kReadQ, q, read_q);
        load_factor(factors(chunk), kReadK, q, read_k);
        last = factors(chunk)[kRise * kRows + kRows - 1];
        Gr.load(chunk_rows(p.go, w.n, w.h, (int64_t)chunk * kRows, Elem<T>::kBytes), g_row, col, p.M,
                min(kRows, w.len - chunk * kRows), q);
    };
    auto load_out = [&](int chunk) {
        if constexpr (kHold) {
#pragma unroll
            for (int i = 0; i < 4 * KE; i++) load_frag(p.qc + (w.key_at + chunk) * kKeys, i, lane, qc[i]);
#pragma unroll
            for (int i = 0; i < 4 * KE; i++) load_frag(p.kc + (w.key_at + chunk) * kKeys, i, lane, kc[i]);
        }
    };
    if (chunks > 0) load_in(chunks - 1), load_t(chunks - 1), load_out(chunks - 1);
    for (int chunk = chunks - 1; chunk >= 0; chunk--) {
        const int64_t at = (w.at + chunk) * p.col_blocks + block;
        const int next = max(chunk - 1, 0);
        {
            float *const to = p.ds + at * (ET * 256) + 4 * lane;
#pragma unroll
            for (int t = 0; t < ET; t++) *(f32x4a *)(to + 256 * t) = S[t];
        }
        f32x4 P[4] = {}, D[4], G[4];
#pragma unroll
        for (int s = 0; s < KE; s++) {
            Frag sf[3];
            cut(S[2 * s], S[2 * s + 1], sf);
#pragma unroll
            for (int t = 0; t < 4; t++)
                P[t] = times<kHold>(kr[t * KE + s], p.kr + (w.key_at + chunk) * kKeys, t * KE + s, lane, sf, P[t]);
        }
        // diag(beta) dU
        f32x4 written = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 4; t++) {
            P[t] *= write[t];
            D[t] = beta[t] * Y[t] + P[t];
            written += Z[t] * P[t];
            P[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        p.written[at * 64 + lane] = (written[0] + written[1]) + (written[2] + written[3]);
        phase();
        load_in(next);
        phase();
        // dE = T^T diag(beta) dU
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag df[3];
            cut(D[2 * s], D[2 * s + 1], df);
#pragma unroll
            for (int t = 0; t < 2 * s + 2; t++) P[t] = product(tf[tt_number(t, s)], df, P[t]);
        }
        store_tiles(p.de + at * (4 * 256) + 4 * lane, P);
        if (p.gv.ptr) {  // (a buffer drops what lies outside)
            const int64_t l0 = (int64_t)chunk * kRows;
            const __amdgpu_buffer_rsrc_t rs = chunk_rows(Operand{p.gv.ptr, p.gv.stride_n, p.gv.stride_h, p.gv.stride_l, 0, 0},
                                                         w.n, w.h, l0, Elem<T>::kBytes);
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int row = 16 * t + 4 * q + r;
                    const uint32_t to = l0 + row < w.len && col < p.M
                                            ? (uint32_t)row * gv_row + (uint32_t)(col * Elem<T>::kBytes) : kOutside;
                    if (Elem<T>::kBytes == 4)
                        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(P[t][r]), rs, to, 0, 0);
                    else
                        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (__bf16)P[t][r]), rs, to, 0, 0);
                }
        }
        settle();
#pragma unroll
        for (int t = 0; t < 4; t++) G[t] = Gr.values(t) * read_q[t], P[t] *= -read_k[t];
#pragma unroll
        for (int t = 0; t < ET; t++) S[t] *= last;
        phase();
        load_t(next);
        phase();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag of[3], ef[3];
            cut(G[2 * s], G[2 * s + 1], of);
#pragma unroll
            for (int t = 0; t < ET; t++)
                S[t] = times<kHold>(qc[2 * t + s], p.qc + (w.key_at + chunk) * kKeys, 2 * t + s, lane, of, S[t]);
            cut(P[2 * s], P[2 * s + 1], ef);
#pragma unroll
            for (int t = 0; t < ET; t++)
                S[t] = times<kHold>(kc[2 * t + s], p.kc + (w.key_at + chunk) * kKeys, 2 * t + s, lane, ef, S[t]);
        }
        phase();
        load_out(next);
        phase();
    }
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
    constexpr int NW = 1;
    const uint32_t groups = (uint32_t)((p.col_blocks + NW - 1) / NW);
    const dim3 grid(((uint32_t)p.N * (uint32_t)p.H + 7) / 8 * 8 * groups);
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
