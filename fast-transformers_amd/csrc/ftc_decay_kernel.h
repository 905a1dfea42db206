// What the kernels of decayed linear attention share: the arguments of a launch.
//
// The attention, per chain (a sequence and a value head) on a state S of E x M in fp32:
//
//   S_t = e^{g_t} S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t
//
// With G_i the sum of g up to i, D_ij = e^{G_i - G_j} for j <= i and s = scale, it and its gradients are one kind of
// scan, out_i = sum over j <= i of D_ij (a_i . b_j) c_j, on four sets of rows, two of them from the last position on:
//
//   o  = scan(q, k, v)              dq = scan(dO, v, k)       state S (of dq: its transpose)
//   dv = reverse scan(k, q, dO)     dk = reverse scan(v, dO, q)       state R = dL/dS
//
// In reverse, the decay between neighbours is that of the later one: row x of a reversed sequence has the log decay
// of the position behind it, and the first one none.  In chunks of 64 rows, G counted from the chunk's start:
//
//   out = diag(e^G) a S + A c,  A_ij = D_ij (a_i . b_j) for j <= i,     S <- e^{G_64} S + b^T diag(e^{G_64 - G}) c
//
// The decays' gradients.  dL/dg_l = X_l, the sum over all pairs (i, j) with j < l <= i of D_ij (q_i . k_j)(dO_i . v_j) s: all
// that crosses from before position l to it or behind.  From one position to the next X loses what position l receives and
// gains what it sends, X_{l+1} = X_l - x_l + y_l with x_l = q_l . dq_l and y_l = k_l . dk_l, both without the diagonal, which
// crosses nothing: with it strong decays would leave X as a small difference of large sums.  So that roundings do not
// add up over a long sequence, both are split into what stays in a chunk, whose sums start at zero in every chunk, and what comes through
// the state, and X at the segments' borders is <S, R> itself (ftc_decay_finish.hip).
#pragma once
#include "ftc_delta_kernel.h"

namespace ftc {
namespace decay {

using delta::Elem;
using delta::f32x4;
using delta::f32x4a;
using delta::Frag;
using delta::kOutside;
using delta::kRows;
using delta::lds_char;
using delta::lds_float;
using delta::Plane;
using delta::RowTile;
using delta::scalar;
using delta::Scalars;
using delta::u32x2;
using delta::u32x2a;
using delta::u32x4;
using mfma::bf16_t;

constexpr int kMaxE = 128;   // the widest key rows
constexpr int kLongest = 1024;  // positions of a segment that has a backward
constexpr int kSlice = 128;  // value rows wider than this are cut into slices, each a chain of its own on the same keys

// Rows as the chains of a launch read them: chain (n, v), v = head * slices + slice, has head v / per of the tensor and, where
// the tensor is one that is cut (`cut` columns a slice, else 0), the columns of its slice.
struct Rows {
    void *ptr;
    int64_t sn, sh, sl;
    int32_t width, per, cut, vec, dtype;  // vec: rows can be accessed 16 bytes at a time
};
struct State {  // (n, h, E, M) fp32, unit stride along M
    float *ptr;
    int64_t sn, sh, sd;
};
struct Task {
    Rows a, b, c, p;  // p: rows whose products with out, without the diagonal, go to dots (or ptr null)
    Rows out;         // ptr null: only the state and the anchors are wanted
    float inter, intra, write;  // factors of what is read from the state, of A, and of what is written to the state
    int32_t reverse, transposed;  // transposed: rows of the state are along M
    float *dots;                // [from the state, altogether][chain][L]
    State first;                // the state handed in
    float *slots;               // states at the segments' borders, [chain][segments + 1][width][slot_rows], or null
};
struct Args {
    Task task[2];
    int32_t tasks;
    int32_t pairs;         // two chains on the same rows of c to a workgroup, whose results are added
    const int64_t *lengths;
    Scalars g;
    int32_t N, H, slices, L, width, slot_rows;  // width: columns of M in a slice (all but the last); slot_rows: E, up to a multiple of 4
    int32_t segments, seg_len, walk;       // walk: a workgroup goes through all segments of its chain (forward)
    State last;            // where the state behind the last chunk goes
    const float *across;   // with anchors: the states S at the borders, against which R is held
    State across_first;    // ... and at the first one
    float *anchors;        // X at the borders, in shares: [chain][segments + 1][shares]
    int32_t shares;
    double *totals;        // the segments' sums of g: [N * H][segments]
};

// 2^x.  (An exponent that is rounded to 24 bits costs |x| 2^-24 of 2^x: as x is not positive, never more than 2^-25.)
__device__ __forceinline__ float power(float x) { return __builtin_amdgcn_exp2f(x); }
// ... of a sum in 64 bits: of its nearest float, and what that leaves
__device__ __forceinline__ float power(float high, float low) { return power(high) * fmaf(low, 0.69314718f, 1.f); }

// depth: columns of a and b; columns: of c; partner: with the products with the rows of p; states: the state alone, of all segments but
// the last on the way, to the border behind each
void decay_scan_f32(const Args &p, int depth, int columns, bool partner, bool states, hipStream_t stream);
void decay_scan_bf16(const Args &p, int depth, int columns, bool partner, bool states, hipStream_t stream);
// columns that a workgroup of such a scan has room for, 16 a wavefront
inline int columns_at_once(int columns) { return columns > 64 ? 128 : 64; }

// ---- behind the scans ----
struct FinishArgs {
    const int64_t *lengths;
    Scalars g, gg;           // gg.ptr null: not wanted
    int32_t N, H, Hk, slices, L, E, segments, seg_len, per_head;
    const float *x, *y;      // the dots of dq and dk
    const float *anchors;
    int32_t shares;
    double *sums;            // per_head: [H][N * segments]
    // shares of the gradients of shared queries or keys, [N][H * slices / every][L][E], and where their sums go
    const float *part[2];
    int32_t every;
    OperandOut sum[2];
};
void decay_borders(const Args &p, const Task &task, hipStream_t stream);
void decay_finish(const FinishArgs &p, hipStream_t stream);
void decay_gather(const FinishArgs &p, hipStream_t stream);

struct StepArgs {
    Operand q, k, v;
    Scalars g;
    const int64_t *lengths;
    State first, last;
    OperandOut out;
    int32_t N, H, Hk, L, E, M;
    float scale;
};
void decay_steps(const StepArgs &p, hipStream_t stream);
bool decay_step_vec(const StepArgs &p);  // whether states are read and written 16 bytes at a time
int64_t decay_step_lanes(int64_t chains, int64_t M, bool vec);

}  // namespace decay
}  // namespace ftc
