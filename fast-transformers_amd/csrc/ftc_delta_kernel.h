// What the kernels of the gated delta rule share: the arguments of a call, the tiles of rows in LDS, the products.
//
// The rule, per chain (a sequence and a value head) on a state S of E x M in fp32:
//
//   S' = exp(g_t) S_{t-1},  z_t = v_t - S'^T k^_t,  S_t = S' + k^_t (beta_t z_t)^T,  o_t = S_t^T q^_t
//
// (k^ = rk k, q^ = rq q: rk, rq the row factors of the normalisation and the scale).  In chunks of 64 positions,
// with G_i the sum of g up to i within the chunk and D_ij = exp(G_i - G_j):
//
//   M_ij = D_ij (k^_i . k^_j) beta_j for j < i,   T = (I + M)^-1                                     (prepare)
//   E = V - diag(e^G) K^ S,   Z = T E,   S <- e^{G_64} S + K^^T diag(beta e^{G_64 - G}) Z            (scan)
//   O = diag(e^G) Q^ S + A diag(beta) Z,   A_ij = D_ij (q^_i . k^_j) for j <= i                     (outputs)
//
// Fidelity of fp32 on the bf16 matrix cores: values of fp32 are cut into three bf16 pieces that add up to them
// exactly, and a product is the sum of the six piece products of order <= 2 (rows that are bf16 have one piece).
// Nothing is rounded to fewer bits before the results are: with the pieces of the state, of T, E and Z cut to one
// the error of bf16 results would grow from 2^-9 to several times that, and final states, gradients of g and beta
// are fp32 results.
//
// Layouts.  v_mfma_f32_16x16x32_bf16: lane (c = lane % 16, q = lane / 16) has, of the result, rows 4 q + r of
// column c.  Two such tiles, rows 0 to 15 and 16 to 31, are the eight values of one k-step of the next product's
// right operand if the left one takes its k in the same order: slots 0 to 3 are k = 4 q + r, slots 4 to 7
// k = 16 + 4 q + r.  So a wavefront that owns 16 columns of the state goes through a chunk's three
// products without an exchange.  What the kernels leave for each other lies in the order of the registers
// ("fragments"): of results, per tile 64 lanes x 4 floats; of left operands, per tile, k-step and piece 64 lanes x 8
// bf16, so that the scan needs neither LDS nor barriers.
#pragma once
#include "ftc_wg_kernel.h"

namespace ftc {
namespace delta {

using mfma::bf16_t;
using mfma::Elem;
using mfma::Frag;
using mfma::lds_char;
using mfma::u32x2;
using mfma::u32x4;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) float lds_float;
typedef float f32x4a __attribute__((ext_vector_type(4), may_alias));
typedef uint32_t u32x2a __attribute__((ext_vector_type(2), may_alias));
typedef uint32_t u32x4a __attribute__((ext_vector_type(4), may_alias));

constexpr int kRows = 64;     // positions of a chunk
constexpr int kCols = 16;     // columns of the state that a wavefront owns
constexpr int kMaxE = 128;    // the widest key rows
constexpr float kNormEps = 1e-6f;

// Row factors of a chunk, 64 floats each, made by the prepare kernel
enum Factor {
    kRise,   // e^{G_i}
    kFall,   // e^{G_64 - G_i}
    kBeta,   // beta_i (0 past the sequence's end)
    kRk,     // 1 / |k_i|, or 1
    kRq,     // scale / |q_i|, or scale
    kRq0,    // 1 / |q_i|, or 1
    kHigh,   // G_i in two floats: its differences are wanted to 24 bits, whatever its size
    kLow,
    kReadK,  // rk e^{G_i}: k_i as it reads the state
    kReadQ,  // rq e^{G_i}
    kWriteK, // rk e^{G_64 - G_i}: as it is written
    kWrite,  // ... times beta_i
    // for the backward, with betas that it can divide by: dbeta is found as dE . Z / beta (all terms of dE have that factor).  Up
    // to 2^-64 in size they count as that there, and such rows of dE for nothing else: their other factors are zero.
    kBetaBack,
    kWriteBack,
    kReadBack,  // kReadK, or 0
    kRkBack,    // kRk, or 0
    kFactors
};
constexpr float kLeastBeta = 0x1p-64f;
constexpr int kSums = 3 * kRows;

struct Scalars {  // one value per position: log decays, beta and their gradients
    void *ptr;
    int64_t sn, sh, sl;
    int32_t dtype;
};

struct DeltaArgs {
    Operand q, k, v;
    Scalars g, b;
    const int64_t *lengths;  // N values, or nullptr
    StateRef initial, final_;
    OperandOut out;
    int32_t N, H, Hk, L, E, M, chunks, col_blocks;  // col_blocks: of 16 columns
    int32_t vec_q, vec_k, vec_v, vec_out, vec_go, vec_gv;  // rows can be read 16 bytes at a time
    int32_t normalize;
    float scale;
    float *factors;          // [chain][chunk][kFactors][64]
    // left operands' fragments, [chain][chunk][number][pieces][64][8]
    uint16_t *t, *tt;        // T and its transpose (may be absent): six with 3 pieces, those not above the diagonal
    uint16_t *kr, *kc, *qc;  // of key chains: rows of k, columns of k and (backward) of q
    // results' fragments
    float *s;                // states before each chunk: [chain][chunk][col block][2 KE tiles][64][4]
    float *z, *o;            // Z and (may be absent) O: [chain][chunk][col block][4 tiles][64][4]
    // backward
    Operand go;
    OperandOut gq, gk, gv;
    Scalars gg, gb;
    StateRef grad_final, grad_initial;
    float *ds;               // the gradient of the state after each chunk, as s
    float *de;               // A^T dO, then dE, as z
    float *dots;             // dO . O of every position, column block by column block: [chain][chunk][col block][64]
    float *sums;             // dE . Z and dE . V of every position, two shares of <S, dS>: [chain][chunk][kSums]
    // few chains: their chunks in segments of seg_chunks (ftc_delta_scan.hip)
    int32_t segments, seg_chunks;
    float *seg;              // what a segment makes of its first state: [chain][segment][col blocks + key blocks][2 KE][64][4]
    float *written;          // shares of what a chunk's keys write of <state, its gradient>: the same, [64 lanes]
};

// ---- rows in LDS ----
// A plane of bf16 pieces: rows of RB bytes (64, 128 or 256) in 8-byte slots, slot p of row r at p ^ key(r).
// The keys (even: 16-byte slots stay whole) keep two patterns free of bank conflicts: 8-byte reads of one
// pair of slots over 16 consecutive rows, and the transposing reads of four slots over eight.
template <int RB>
struct Plane {
    static constexpr int kBytes = kRows * RB;
    __device__ static __forceinline__ int key(int r) {
        if (RB == 64) return (((r >> 2) & 1) << 2) | (((r >> 3) & 1) << 1);
        if (RB == 128) return (((r >> 1) & 3) << 2) | (((r >> 3) & 1) << 1);
        return ((r & 7) << 2) | (((r >> 3) & 1) << 1);
    }
    __device__ static __forceinline__ int addr(int row, int slot) { return row * RB + ((slot ^ key(row)) << 3); }
    // rows 16 t .. of the operand, k-step s (32 values): lane's row c, k = 4 q .. and 16 + 4 q ..
    __device__ static __forceinline__ Frag rows(const lds_char *p, int t, int s, int c, int q) {
        const u32x2 lo = *(const __attribute__((address_space(3))) u32x2a *)(p + addr(16 * t + c, 8 * s + q));
        const u32x2 hi = *(const __attribute__((address_space(3))) u32x2a *)(p + addr(16 * t + c, 8 * s + 4 + q));
        return Frag{{lo.x, lo.y, hi.x, hi.y}};
    }
    // columns 16 t .. as the operand's rows, rows 32 s .. of the plane as its k
    __device__ static __forceinline__ Frag columns(const lds_char *p, int t, int s, int c, int q) {
        const int at = addr(32 * s + 4 * q + (c >> 2), 4 * t + (c & 3));
        return mfma::lds_frag_tr(p + at, p + at + 16 * RB);
    }
};

__device__ __forceinline__ f32x4 mfma16(const Frag &a, const Frag &b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mfma::bf16x8, a),
                                                   __builtin_bit_cast(mfma::bf16x8, b), c, 0, 0, 0);
}
// fp32 values as they are: lane's a is row c of column q, b row q of column c
__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 acc) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma4(const f32x4 &a, const f32x4 &b, f32x4 acc) {
#pragma unroll
    for (int r = 0; r < 4; r++) acc = mfma4(a[r], b[r], acc);
    return acc;
}
// acc += A B over the piece products of order <= 2, smallest first
template <int NA, int NB>
__device__ __forceinline__ f32x4 product(const Frag (&a)[NA], const Frag (&b)[NB], f32x4 acc) {
#pragma unroll
    for (int order = 2; order >= 0; order--)
#pragma unroll
        for (int pa = 0; pa < NA; pa++) {
            const int pb = order - pa;
            if (pb >= 0 && pb < NB) acc = mfma16(a[pa], b[pb], acc);
        }
    return acc;
}
// ... of several tiles by one right operand, a piece product of every tile after the other: each waits for its
// tile's last one, which has had the others' time
template <int FROM, int TILES, int NA, int NB>
__device__ __forceinline__ void products(const Frag (&a)[TILES][NA], const Frag (&b)[NB], f32x4 (&acc)[TILES]) {
#pragma unroll
    for (int order = 2; order >= 0; order--)
#pragma unroll
        for (int pa = 0; pa < NA; pa++) {
            const int pb = order - pa;
            if (pb >= 0 && pb < NB)
#pragma unroll
                for (int t = FROM; t < TILES; t++) acc[t] = mfma16(a[t][pa], b[pb], acc[t]);
        }
}
// Lets the last products' results arrive before a branch.  The compiler counts the instructions between a matrix
// product and the first use of its result, but where a branch skips a block it counts those of the block on the path
// without them too (seen in a listing: a result read two instructions after its product, and wrong rows).  Where it has to
// stand is checked on the listings of all kernels, by tests/test_matrix_results.py.
__device__ __forceinline__ void settle() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15");
    __builtin_amdgcn_sched_barrier(0);
}
// two tiles of a result -> the k-step that they are for the next product
__device__ __forceinline__ void cut(const f32x4 &lo, const f32x4 &hi, Frag (&f)[3]) {
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            uint32_t o[3];
            const f32x4 &x = h ? hi : lo;
            mfma::split_pair_under_mfma(x[2 * j], x[2 * j + 1], o);
#pragma unroll
            for (int p = 0; p < 3; p++) f[p].w[2 * h + j] = o[p];
        }
}
// values that were bf16 to begin with: one piece
__device__ __forceinline__ void cut(const f32x4 &lo, const f32x4 &hi, Frag (&f)[1]) {
    f[0].w[0] = mfma::pack_hi16(lo[0], lo[1]), f[0].w[1] = mfma::pack_hi16(lo[2], lo[3]);
    f[0].w[2] = mfma::pack_hi16(hi[0], hi[1]), f[0].w[3] = mfma::pack_hi16(hi[2], hi[3]);
}

// ---- rows from memory ----
constexpr uint32_t kOutside = 0x80000000u;  // an offset that no buffer reaches: reads as zero

__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A chunk's rows of one chain.  Offsets within it stay below 2 GiB (the strides are checked for that); the
// chunk's own place is in the 64-bit base.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t chunk_rows(const Operand &o, int64_t n, int64_t h, int64_t l0,
                                                            int bytes) {
    const uint64_t at = (uint64_t)o.ptr + (uint64_t)((n * o.stride_n + h * o.stride_h + l0 * o.stride_l) * bytes);
    // (the same in every lane; the compiler, which has made it from a division, would try the lanes one by one)
    const char *base = (const char *)(((uint64_t)(uint32_t)scalar((int)(at >> 32)) << 32) | (uint32_t)scalar((int)(uint32_t)at));
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, 0x7fffffff, mfma::kRsrcFlags);
}

template <typename T>
__device__ __forceinline__ float load_one(__amdgpu_buffer_rsrc_t rs, uint32_t offset);
template <>
__device__ __forceinline__ float load_one<float>(__amdgpu_buffer_rsrc_t rs, uint32_t offset) {
    return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, offset, 0, 0));
}
template <>
__device__ __forceinline__ float load_one<bf16_t>(__amdgpu_buffer_rsrc_t rs, uint32_t offset) {
    return bf16_to_f32(__builtin_amdgcn_raw_buffer_load_b16(rs, offset, 0, 0));
}

// 64 rows of up to COLS values (zeros beyond the width and the last valid row) by NT threads: into registers, then
// into LDS planes.  Unit u: eight values of row u / (COLS / 8).
template <typename T, int COLS, int NT>
struct RowTile {
    static constexpr int kUnits = kRows * COLS / 8, kPer = kUnits / NT, kAcross = COLS / 8;
    static constexpr int kPieces = Elem<T>::kPieces, kBytes = Elem<T>::kBytes;
    u32x4 r[kPer][kBytes / 2];

    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t row_bytes, int width, int valid, bool vec,
                                         int tid) {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int u = tid + NT * i, row = u / kAcross, col = 8 * (u % kAcross);
            const uint32_t base = (uint32_t)row * row_bytes + (uint32_t)(col * kBytes);
            if (vec) {
#pragma unroll
                for (int j = 0; j < kBytes / 2; j++)  // (fp32: widths are multiples of 4, bf16: of 8)
                    r[i][j] = __builtin_amdgcn_raw_buffer_load_b128(
                        rs, row < valid && col + 4 * j < width ? base + 16 * j : kOutside, 0, 0);
            } else if (kBytes == 4) {
#pragma unroll
                for (int x = 0; x < 8; x++)
                    r[i][(x / 4) % (kBytes / 2)][x % 4] = __builtin_amdgcn_raw_buffer_load_b32(
                        rs, row < valid && col + x < width ? base + 4 * x : kOutside, 0, 0);
            } else {
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const uint32_t lo = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(
                        rs, row < valid && col + 2 * x < width ? base + 4 * x : kOutside, 0, 0);
                    const uint32_t hi = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(
                        rs, row < valid && col + 2 * x + 1 < width ? base + 4 * x + 2 : kOutside, 0, 0);
                    r[i][0][x] = lo | (hi << 16);
                }
            }
        }
    }
    __device__ __forceinline__ float value(int i, int x) const {  // value x of the lane's unit i
        if (kBytes == 4) return __uint_as_float(r[i][(x / 4) % (kBytes / 2)][x % 4]);
        return __uint_as_float(x % 2 ? r[i][0][x / 2] & 0xffff0000u : r[i][0][x / 2] << 16);
    }
    template <int RB>
    __device__ __forceinline__ void store(lds_char *planes, int tid) const {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int u = tid + NT * i, row = u / kAcross, slot = 2 * (u % kAcross);
            lds_char *const to = planes + Plane<RB>::addr(row, slot);
            if (kPieces == 1) {
                *(__attribute__((address_space(3))) u32x4a *)to = r[i][0];
            } else {
                u32x4 o[3];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    uint32_t p[3];
                    mfma::split_pair_under_mfma(value(i, 2 * x), value(i, 2 * x + 1), p);
                    o[0][x] = p[0], o[1][x] = p[1], o[2][x] = p[2];
                }
#pragma unroll
                for (int p = 0; p < 3; p++)
                    *(__attribute__((address_space(3))) u32x4a *)(to + p * Plane<RB>::kBytes) = o[p];
            }
        }
    }
};

// The pieces of a fragment, read from planes one after the other
template <int RB, int PIECES>
__device__ __forceinline__ void rows_of(const lds_char *planes, int t, int s, int c, int q, Frag (&f)[PIECES]) {
#pragma unroll
    for (int p = 0; p < PIECES; p++) f[p] = Plane<RB>::rows(planes + p * Plane<RB>::kBytes, t, s, c, q);
}
template <int RB, int PIECES>
__device__ __forceinline__ void columns_of(const lds_char *planes, int t, int s, int c, int q, Frag (&f)[PIECES],
                                           int plane_bytes = Plane<RB>::kBytes) {
#pragma unroll
    for (int p = 0; p < PIECES; p++) f[p] = Plane<RB>::columns(planes + p * plane_bytes, t, s, c, q);
}

// Two values -> two bf16, rounded to nearest
__device__ __forceinline__ uint32_t to_bf16(float x0, float x1) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x0, x1}, bf16x2));
}
// Four values of consecutive columns of a row -> the planes of their three pieces
__device__ __forceinline__ void store_pieces(lds_char *to, int plane_bytes, const f32x4 &x) {
    uint32_t a[3], b[3];
    mfma::split_pair_under_mfma(x[0], x[1], a);
    mfma::split_pair_under_mfma(x[2], x[3], b);
#pragma unroll
    for (int p = 0; p < 3; p++)
        *(__attribute__((address_space(3))) u32x2a *)(to + p * plane_bytes) = u32x2{a[p], b[p]};
}

// ---- left operands' fragments in memory ----
template <int PIECES>
__device__ __forceinline__ void load_frag(const uint16_t *from, int number, int lane, Frag (&f)[PIECES]) {
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
        const u32x4 r = *(const u32x4a *)(from + (number * PIECES + p) * 512 + 8 * lane);
        f[p] = Frag{{r.x, r.y, r.z, r.w}};
    }
}
template <int PIECES>
__device__ __forceinline__ void store_frag(uint16_t *to, int number, int lane, const Frag (&f)[PIECES]) {
#pragma unroll
    for (int p = 0; p < PIECES; p++)
        *(u32x4a *)(to + (number * PIECES + p) * 512 + 8 * lane) = u32x4{f[p].w[0], f[p].w[1], f[p].w[2], f[p].w[3]};
}
// T: row tile t has k-steps 0 .. t / 2; its transpose k-steps t / 2 .. 1
constexpr int kTFrags = 6;
__device__ __forceinline__ constexpr int t_number(int t, int s) { return t < 2 ? t : 2 * t - 2 + s; }
__device__ __forceinline__ constexpr int tt_number(int t, int s) { return t < 2 ? 2 * t + s : t + 2; }

// ---- places ----
struct Where {
    int32_t chain, n, h, hk, chunk, len, valid;  // len: positions of the sequence; valid: of them in this chunk
    int64_t at, key_at;                          // chain * chunks + chunk, and of the key head's chain
};
__device__ __forceinline__ int sequence_length(const DeltaArgs &p, int n) {
    if (!p.lengths) return p.L;
    const int64_t len = p.lengths[n];
    return (int)(len < 0 ? 0 : len > p.L ? p.L : len);
}
__device__ __forceinline__ Where where_of(const DeltaArgs &p, int chain, int chunk) {
    Where w;
    w.chain = scalar(chain), w.chunk = scalar(chunk);
    w.n = scalar(w.chain / p.H), w.h = w.chain - w.n * p.H, w.hk = scalar(w.h / (p.H / p.Hk));
    w.len = scalar(sequence_length(p, w.n));
    const int left = w.len - w.chunk * kRows;
    w.valid = left < 0 ? 0 : left > kRows ? kRows : left;
    w.at = (int64_t)w.chain * p.chunks + w.chunk;
    w.key_at = ((int64_t)w.n * p.Hk + w.hk) * p.chunks + w.chunk;
    return w;
}
__device__ __forceinline__ int chunks_of(int len) { return (len + kRows - 1) / kRows; }

// sum over the 16 lanes of a row of lanes, in every one of them
__device__ __forceinline__ float sum16(float x) {
#define FTC_ROR(N) \
    x += __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x120 + (N), 0xf, 0xf, false));
    FTC_ROR(8) FTC_ROR(4) FTC_ROR(2) FTC_ROR(1)
#undef FTC_ROR
    return x;
}

// Launchers (one translation unit each); `pieces` by the rows' element type
int delta_prepare(const DeltaArgs &p, bool bf16, hipStream_t stream);
int delta_scan(const DeltaArgs &p, bool bf16, hipStream_t stream);
int delta_outputs(const DeltaArgs &p, bool bf16, hipStream_t stream);
int delta_pull(const DeltaArgs &p, bool bf16, hipStream_t stream);           // A^T dO
int delta_scan_back(const DeltaArgs &p, bool bf16, hipStream_t stream);
int delta_gradients(const DeltaArgs &p, bool bf16, hipStream_t stream);
int delta_steps(const DeltaArgs &p, hipStream_t stream);                        // position by position

// How many wavefronts of a scan share its operands (first: in the launch that makes the segments' maps)
int delta_scan_shared_by(const DeltaArgs &p, bool bf16, bool first);

}  // namespace delta
}  // namespace ftc
