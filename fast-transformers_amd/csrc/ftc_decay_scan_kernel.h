// Decayed linear attention: the scan of one chain's chunks, forward and reverse.  Formulas: ftc_decay_kernel.h, layouts of the
// tiles and fragments: ftc_delta_kernel.h.
//
// A workgroup walks the chunks of one segment of a chain (or of all of them).  A wavefront owns 16 columns of the result
// and of the state, which stays in its registers from chunk to chunk; A is made once for all, in LDS, where the rows of a
// were.  The next chunk's rows are on their way meanwhile.  The result is made transposed, state and c from the left, so that a lane
// has four columns of one row: they are stored at once, and its products with other rows need two exchanges a row.
//
// Pieces.  Products of rows are exact on the bf16 matrix cores, of fp32 rows in three pieces.  The state that is written
// takes three pieces of what it adds, and so does whatever becomes a gradient of the decays: those are results of fp32.
// What only becomes a result of bf16 takes two (to 2^-17, where its own rounding is 2^-8): 128 chains of 4096 x 128 x 128, bf16, take
// 225 us forward with two and 238 with three.
//
// What bounds it: vector instructions (cuts into pieces, factors, addresses) and what a chunk's phases wait for each other, not memory.  A
// launch of that size takes 138 us (403 MB of rows, 2.9 TB/s; vector instructions 57 % of a SIMD's cycles, matrix instructions 36 %, LDS 33 %
// of a compute unit's), one that makes the states alone 60 (201 MB), the queries' and keys' gradients together 360.  (So they take in a row of passes;
// the first ones, before the card is at its clocks, take up to 30 % longer, in as many cycles.)  80 chains of 1000 x 64 x 64,
// fp32: 32, 15 and 63 us, 480 workgroups (of four wavefronts) that walk three chunks each: 5.7 us a chunk by themselves, 9 for two of them.
// Figures that stand side by side in these comments are of one card, taken in turn.
//
// Tried: wavefronts in two groups, one for the state and one for A, for fp32 rows (52 us forward as before, 227 with the gradients
// instead of 182: registers); operands of two columns of wavefronts read once (spills); first remainders of pieces as dot products (they have
// to be copied first: 830 us instead of 800 for the whole of the first case), all remainders as subtractions (834).
#pragma once
#include "ftc_decay_kernel.h"

namespace ftc {
namespace decay {
namespace {

enum Mode { kPlain, kPartner, kStates };  // results; results and their products with other rows; the state alone

using delta::product;
using delta::settle;

constexpr int kAPlane = Plane<128>::kBytes;

// Two values in NP pieces: three that add up to them, or two, the second rounded to nearest.  (A remainder is one instruction here, which
// waits for the wavefront's own products; the others' time fills that, and what bounds the scan is how many are issued.)
template <int NP>
__device__ __forceinline__ void cut_pair(float x0, float x1, uint32_t (&o)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; i++) {
        o[i] = NP == 2 && i == 1 ? delta::to_bf16(x0, x1) : mfma::pack_hi16(x0, x1);
        if (i == 0) {
            x0 -= __uint_as_float(__float_as_uint(x0) & 0xffff0000u), x1 -= __uint_as_float(__float_as_uint(x1) & 0xffff0000u);
        } else if (i + 1 < NP) {
            x0 = mfma::minus_piece(x0, o[i], mfma::minus_one_even());
            x1 = mfma::minus_piece(x1, o[i], mfma::minus_one_odd());
        }
    }
}
// Two tiles of a result as the next product's operand
template <int NP>
__device__ __forceinline__ void cut(const f32x4 &lo, const f32x4 &hi, Frag (&f)[NP]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const f32x4 &x = j < 2 ? lo : hi;
        uint32_t o[NP];
        cut_pair<NP>(x[2 * (j % 2)], x[2 * (j % 2) + 1], o);
#pragma unroll
        for (int i = 0; i < NP; i++) f[i].w[j] = o[i];
    }
}
template <int NP>
__device__ __forceinline__ void put_pieces(lds_char *to, const f32x4 &x) {
    uint32_t a[NP], b[NP];
    cut_pair<NP>(x[0], x[1], a);
    cut_pair<NP>(x[2], x[3], b);
#pragma unroll
    for (int i = 0; i < NP; i++) *(__attribute__((address_space(3))) u32x2a *)(to + i * kAPlane) = u32x2{a[i], b[i]};
}

// Planes of rows that are only read as rows, a and A: slots lie so that an operand's two groups of four, 4 q and 16 + 4 q of 32, are
// side by side, and are read at once.  (Of b, which is read as columns too, they would meet in the same banks.)  The 16-byte units of
// row r lie at their number ^ key(r): sixteen lanes of such a read, whether they are those of q or rows 0 to 3 and 12 to 15 of q and 4 to 11
// of q + 1, have all 64 banks.  (With the keys of rows that are read 8 bytes at a time, a third of LDS's time went to conflicts.)
template <int RB>
struct Paired {
    static_assert(RB == 128 || RB == 256, "");
    __device__ static __forceinline__ int key(int row) { return RB == 256 ? row & 15 : row >> 1 & 7; }
    // four values of a row, from column 4 slot on
    __device__ static __forceinline__ int addr(int row, int slot) {
        return row * RB + (((slot >> 3 << 2 | (slot & 3)) ^ key(row)) << 4 | (slot & 4) << 1);
    }
    // (keys are the same 16 rows on, and k-steps change bits of an address that nothing else changes)
    template <int PIECES>
    __device__ static __forceinline__ void rows_of(const lds_char *planes, int t, int s, int c, int q, Frag (&f)[PIECES]) {
        const int at = (c * RB + ((q ^ key(c)) << 4)) ^ s << 6;
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const u32x4 x = *(const __attribute__((address_space(3))) delta::u32x4a *)(planes + at + i * Plane<RB>::kBytes + 16 * RB * t);
            f[i] = Frag{{x.x, x.y, x.z, x.w}};
        }
    }
};
// Columns of b or c as an operand's rows, as Plane::columns has them
template <int RB, int PIECES>
__device__ __forceinline__ void columns_of(const lds_char *planes, int t, int s, int c, int q, Frag (&f)[PIECES]) {
    const int row = 4 * q + (c >> 2), at = (row * RB + (((c & 3) ^ Plane<RB>::key(row)) << 3)) ^ t << 5;
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        const lds_char *const from = planes + at + i * Plane<RB>::kBytes + 32 * RB * s;
        f[i] = mfma::lds_frag_tr(from, from + 16 * RB);
    }
}
// Rows of b: two reads of an operand, kept apart (two rows' reads in one would leave its halves in registers that have to be moved)
template <int RB, int PIECES>
__device__ __forceinline__ void rows_apart(const lds_char *planes, int t, int s, int c, int q, Frag (&f)[PIECES]) {
    typedef const volatile __attribute__((address_space(3))) uint64_t *At;
    const int first = (c * RB + ((q ^ Plane<RB>::key(c)) << 3)) ^ s << 6;
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        const lds_char *const at = planes + i * Plane<RB>::kBytes + 16 * RB * t;
        const uint64_t lo = *(At)(at + first), hi = *(At)(at + (first ^ 32));
        f[i] = Frag{{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)}};
    }
}
__device__ __forceinline__ f32x4 widen(const u32x2 &x) {  // four bf16
    return f32x4{__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xffff0000u)};
}

// A chunk on the way: its lowest position, and how many it has
struct Chunk {
    int base, valid;
};

// N words at any address that bf16 may have
template <int N>
using Any = uint32_t __attribute__((ext_vector_type(N), aligned(2), may_alias));
// Eight values (kB bytes each) or four, so many places down, zeros behind
template <int kB, int WORDS4>
__device__ __forceinline__ void move_down(u32x4 (&x)[WORDS4], int by) {
    constexpr int kWords = 4 * WORDS4;
    uint32_t w[kWords + 1];
#pragma unroll
    for (int i = 0; i < kWords; i++) w[i] = x[i / 4][i % 4];
    w[kWords] = 0u;
    const int words = kB == 4 ? by : by >> 1;
#pragma unroll
    for (int bit = 4; bit >= 1; bit /= 2)
#pragma unroll
        for (int i = 0; i < kWords; i++) {
            const uint32_t from = i + bit < kWords ? w[(i + bit) % kWords] : 0u, own = w[i];
            w[i] = words & bit ? from : own;
        }
    if (kB == 2)
#pragma unroll
        for (int i = 0; i < kWords; i++) {
            const uint32_t pair = w[i] >> 16 | w[i + 1] << 16, own = w[i];
            w[i] = by & 1 ? pair : own;
        }
#pragma unroll
    for (int i = 0; i < kWords; i++) x[i / 4][i % 4] = w[i];
}

// Rows of a chunk, from the last one on where they are wanted in reverse.  VEC: all of a launch's rows lie on 16 bytes and have whole
// ones.  (The other way works for any: 128 chains of 4096 x 128 x 128, bf16, 257 us forward for 236; 80 of 1000 x 64 x 64, fp32, with
// gradients 194 for 175; 64 of 2048 x 128 x 64, fp32, 143 for 127.)
template <typename T, int COLS, int NT, bool VEC>
struct Tile : RowTile<T, COLS, NT> {
    using Base = RowTile<T, COLS, NT>;
    static constexpr int kB = Base::kBytes, kStep = NT / Base::kAcross;  // rows between a lane's units
    __device__ __forceinline__ void fetch(const char *rows, uint32_t row_bytes, int width, int valid, int tid, bool flip) {
        const int row0 = tid / Base::kAcross, col = 8 * (tid % Base::kAcross);
        if constexpr (VEC) {  // (fp32: widths are multiples of 4, bf16: of 8)
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)rows, 0, 0x7fffffff, mfma::kRsrcFlags);
            const uint32_t first = (uint32_t)(flip ? valid - 1 - row0 : row0) * row_bytes + (uint32_t)(col * kB);
            const uint32_t step = flip ? 0u - kStep * row_bytes : kStep * row_bytes;
#pragma unroll
            for (int i = 0; i < Base::kPer; i++)
#pragma unroll
                for (int j = 0; j < kB / 2; j++)
                    this->r[i][j] = __builtin_amdgcn_raw_buffer_load_b128(
                        rs, row0 + kStep * i < valid && col + 4 * j < width ? first + i * step + 16 * j : kOutside, 0, 0);
        } else {
            // eight values at any address; where the row ends among them its last eight, moved to their places
            const int by = max(0, col + 8 - width);
#pragma unroll
            for (int i = 0; i < Base::kPer; i++) {
                const int row = row0 + kStep * i;
                u32x4 x[kB / 2];
#pragma unroll
                for (int j = 0; j < kB / 2; j++) x[j] = u32x4{0u, 0u, 0u, 0u};
                if (row < valid && col < width) {
                    const char *const at = rows + (uint32_t)((flip ? valid - 1 - row : row) * row_bytes);
                    if (width >= 8) {
#pragma unroll
                        for (int j = 0; j < kB / 2; j++) x[j] = *(const Any<4> *)(at + (col - by) * kB + 16 * j);
                        if (by) move_down<kB>(x, by);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; k++)
                            if (col + k < width) {
                                if constexpr (kB == 4) x[(k / 4) % (kB / 2)][k % 4] = ((const uint32_t *)at)[k];
                                else x[0][k / 2] |= (uint32_t)((const uint16_t *)at)[k] << (16 * (k % 2));
                            }
                    }
                }
#pragma unroll
                for (int j = 0; j < kB / 2; j++) this->r[i][j] = x[j];
            }
        }
    }
    // into planes that are read in pairs
    template <int RB>
    __device__ __forceinline__ void store_paired(lds_char *planes, int tid) const {
#pragma unroll
        for (int i = 0; i < Base::kPer; i++) {
            const int row = tid / Base::kAcross + kStep * i, slot = 2 * (tid % Base::kAcross);
#pragma unroll
            for (int half = 0; half < 2; half++) {
                lds_char *const to = planes + Paired<RB>::addr(row, slot + half);
                if constexpr (Base::kPieces == 1) {
                    *(__attribute__((address_space(3))) u32x2a *)to = u32x2{this->r[i][0][2 * half], this->r[i][0][2 * half + 1]};
                } else {
                    uint32_t a[3], b[3];
                    cut_pair<3>(this->value(i, 4 * half), this->value(i, 4 * half + 1), a);
                    cut_pair<3>(this->value(i, 4 * half + 2), this->value(i, 4 * half + 3), b);
#pragma unroll
                    for (int k = 0; k < 3; k++)
                        *(__attribute__((address_space(3))) u32x2a *)(to + k * Plane<RB>::kBytes) = u32x2{a[k], b[k]};
                }
            }
        }
    }
    // fp32 rows as they are, `stride` floats apart
    __device__ __forceinline__ void put(lds_float *to, int stride, int tid) const {
#pragma unroll
        for (int i = 0; i < Base::kPer; i++)
#pragma unroll
            for (int j = 0; j < kB / 2; j++)
                *(__attribute__((address_space(3))) delta::u32x4a *)(to + (tid / Base::kAcross + kStep * i) * stride + 8 * (tid % Base::kAcross) + 4 * j) =
                    this->r[i][j];
    }
};

struct Chain {
    int at, n, v, slice, head, len;  // at: n * heads * slices + v
};
__device__ __forceinline__ Chain chain_of(const Args &p, int at) {
    Chain w;
    w.at = scalar(at);
    const int per = p.H * p.slices;
    w.n = scalar(w.at / per), w.v = w.at - w.n * per;
    w.head = scalar(w.v / p.slices), w.slice = w.v - w.head * p.slices;
    int64_t len = p.lengths ? p.lengths[w.n] : p.L;
    len = len < 0 ? 0 : len > p.L ? p.L : len;
    w.len = scalar((int)len);
    return w;
}
__device__ __forceinline__ char *address(const void *ptr, int64_t bytes) {
    const uint64_t at = (uint64_t)ptr + (uint64_t)bytes;
    return (char *)(((uint64_t)(uint32_t)scalar((int)(at >> 32)) << 32) | (uint32_t)scalar((int)(uint32_t)at));
}
__device__ __forceinline__ int width_of(const Rows &o, const Chain &w) {
    return o.cut ? min(o.cut, o.width - o.cut * w.slice) : o.width;
}
// A chain's rows, made once; offsets within a chunk stay below 2 GiB (the strides are checked for that)
struct From {
    char *ptr;
    uint32_t row_bytes;
    __device__ __forceinline__ char *at(int l) const { return ptr + (uint64_t)row_bytes * (uint32_t)l; }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(int l) const {
        return __builtin_amdgcn_make_buffer_rsrc(at(l), 0, 0x7fffffff, mfma::kRsrcFlags);
    }
};
__device__ __forceinline__ From rows_from(const Rows &o, const Chain &w, int bytes) {
    const int64_t at = w.n * o.sn + (int64_t)(o.per > 0 ? w.v / o.per : 0) * o.sh + (o.cut ? o.cut * w.slice : 0);
    return From{address(o.ptr, at * bytes), (uint32_t)o.sl * bytes};
}

// Factors of a chunk's rows, in LDS
enum Factor { kHigh, kLow, kRise, kFall, kFactors };  // G / ln 2 in two floats, inter e^G, write e^{G_64 - G}
// Inclusive sums over the lanes of a wavefront, in 64 bits, without LDS
template <int CONTROL, int ROWS>
__device__ __forceinline__ double moved(double x) {  // 0 where nothing comes from
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CONTROL, ROWS, 0xf, false),
                   hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CONTROL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double sums_so_far(double x) {
    x += moved<0x111, 0xf>(x);  // one lane up in its row of 16, two, four, eight
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    x += moved<0x118, 0xf>(x);
    x += moved<0x142, 0xa>(x);  // a row's last lane to the next row's, in rows 1 and 3
    x += moved<0x143, 0xc>(x);  // lane 31 to rows 2 and 3
    return x;
}
__device__ __forceinline__ double of_last_lane(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), 63) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 63));
}

// A number of the lane's anew: addresses made of it belong to the phase behind (those of all phases, held through the loop over
// chunks, would not leave registers for the products)
template <int MOST>
__device__ __forceinline__ int renewed(int x) {
    asm volatile("" : "+v"(x));
    __builtin_assume(x >= 0 && x < MOST);
    return x;
}

// Scans that are held to 128 registers, for sixteen wavefronts a compute unit, and to the order in which they are written.  (128 chains of
// 2048 x 128 x 128, with gradients: 500 us, 517 without.)
template <typename T, int KE, int WAVES, int MODE, int HEADS>
constexpr bool kTight = Elem<T>::kPieces == 1 && KE == 4 && WAVES == 8 && MODE == kPartner && HEADS == 1;

// Wavefronts that a SIMD is to hold: four of a workgroup alone where their LDS leaves no room for a second one
template <typename T, int KE, int WAVES, int MODE, int HEADS>
constexpr int kSide = kTight<T, KE, WAVES, MODE, HEADS> ? 4 : Elem<T>::kPieces == 3 && KE == 4 && WAVES == 4 && MODE != kStates ? 1 : 2;

// HEADS: 2 for the gradients of queries or keys that an even number of chains share (bf16): a workgroup takes two chains of one key
// head, WAVES wavefronts each, on the same rows of c, and adds their results before they are stored.  (The other way is to store them in
// fp32 and add them in a launch of its own.  8 sequences of 4096 with 16 heads on 8 key heads, with gradients: 64 x 64 462 us, the other way 485;
// 128 x 64 585, 742; 64 x 128 590, 657; 128 x 128 824, 974.  Few chains: 4 heads on one, 1024 positions, 114, 110.)
template <typename T, int KE, int WAVES, int MODE, bool VEC, int HEADS>
__global__ __launch_bounds__(64 * WAVES * HEADS, (kSide<T, KE, WAVES, MODE, HEADS>)) void decay_scan_kernel(Args p) {
    static_assert(HEADS == 1 || (MODE == kPartner && Elem<T>::kPieces == 1), "results are added where A does not lie");
    constexpr int PIECES = Elem<T>::kPieces, NT = 64 * WAVES, kB = Elem<T>::kBytes;
    constexpr int RB = 64 * KE, ET = 2 * KE, NP = PIECES == 3 || MODE == kPartner ? 3 : 2;
    constexpr int COLS = 16 * WAVES;               // columns of the workgroup
    constexpr bool kHeld = kTight<T, KE, WAVES, MODE, HEADS>;
    constexpr bool kNarrow = PIECES == 1;          // bf16 rows of c as they are, fp32 ones as floats
    constexpr int RC = kNarrow ? 2 * COLS : 64, kStrideC = COLS + 4, kRowsC = kNarrow ? kRows * RC : kRows * kStrideC * 4;
    constexpr int kRowsA = PIECES * Plane<RB>::kBytes;
    // (A of fp32 rows lies where those of a were: two workgroups fit a compute unit)
    constexpr bool kOver = PIECES == 3;
    constexpr int kTwo = HEADS == 2 ? WAVES * 2 * 1024 : 0;  // two tiles of every wavefront's result
    constexpr int kRoom = kRowsA > kTwo ? kRowsA : kTwo;
    constexpr int kA = MODE == kStates ? 0 : !kOver ? kRoom + NP * kAPlane : kRowsA > NP * kAPlane ? kRowsA : NP * kAPlane;
    __shared__ __align__(16) char mem[HEADS * (kA + kRowsA) + kRowsC];
    __shared__ __align__(16) float f_mems[HEADS][2][kFactors * kRows];
    __shared__ float diag_mems[HEADS][MODE == kPartner ? kRows : 1];
    __shared__ float dot_mems[HEADS][MODE == kPartner ? 2 * WAVES * kRows : 1];
    const int lane = threadIdx.x & 63, half = HEADS == 1 ? 0 : scalar(threadIdx.x / NT), wave = scalar(threadIdx.x >> 6) - half * WAVES;
    lds_char *const ap = (lds_char *)mem + half * (kA + kRowsA), *const Ap = ap + (kOver ? 0 : kRoom), *const bp = ap + kA,
                   *const cp = (lds_char *)mem + HEADS * (kA + kRowsA);
    float(&f_mem)[2][kFactors * kRows] = f_mems[half];
    float *const diag_mem = diag_mems[half], *const dot_mem = dot_mems[half];

    int c = lane & 15, q = lane >> 4;
    auto renew = [&]() {
        if (kHeld) __builtin_amdgcn_sched_barrier(0);
        c = renewed<16>(c), q = renewed<4>(q);
    };
    // workgroups go to the eight dies in turn: those that share rows to the same
    const int die = (int)(blockIdx.x & 7), turn = scalar((int)(blockIdx.x >> 3));
    const int unit = scalar((turn / p.tasks) * 8 + die);
    const Task &task = p.task[turn % p.tasks];
    const bool flip = task.reverse;
    // (the state alone: of all segments but the last on the way)
    const int count = MODE == kStates ? p.segments - 1 : p.walk ? 1 : p.segments;
    const int at = scalar(unit / count) * HEADS + half, part = unit - at / HEADS * count;
    if (at >= p.N * p.H * p.slices) return;
    const Chain w = chain_of(p, at);
    const int first_seg = p.walk ? 0 : MODE == kStates && flip ? part + 1 : part, segs = p.walk ? p.segments : 1;

    const int width_a = width_of(MODE == kStates ? task.b : task.a, w), width_c = width_of(task.c, w);
    const int mine = wave * 16;  // the wavefront's first column of c
    const int64_t slot_size = (int64_t)p.slot_rows * p.width;
    float *const slots = task.slots ? task.slots + (int64_t)w.at * (p.segments + 1) * slot_size : nullptr;

    auto segment = [&](int seg, int &start, int &end) {
        start = seg * p.seg_len;
        const int64_t stop = min((int64_t)start + p.seg_len, (int64_t)p.L);
        end = (int)min(stop, (int64_t)w.len);
    };
    auto chunks_in = [&](int seg) {
        int start, end;
        segment(seg, start, end);
        return end > start ? (end - start + kRows - 1) / kRows : 0;
    };
    auto chunk_at = [&](int seg, int x) {
        int start, end;
        segment(seg, start, end);
        const int base = start + kRows * (flip ? (end - start - 1) / kRows - x : x);
        return Chunk{base, min(kRows, end - base)};
    };

    // ---- rows on their way ----
    Tile<T, 32 * KE, NT, VEC> a_tile, b_tile;
    Tile<T, COLS, NT * HEADS, VEC> c_tile;
    using Quad = typename std::conditional<kNarrow, u32x2, u32x4>::type;
    Quad p_own[4];         // four columns of row 16 t + c
    float g_next = 0.f;
    const From a_from = rows_from(task.a, w, kB), b_from = rows_from(task.b, w, kB), c_from = rows_from(task.c, w, kB),
               p_from = rows_from(task.p, w, kB);
    const bool partner = MODE == kPartner && task.p.ptr;
    const bool narrow = kNarrow && task.out.dtype == FTC_BF16;  // (shares of gradients of bf16 are fp32)
    const int bytes = narrow ? 2 : 4;
    const From out_to = rows_from(task.out, w, bytes);
    const char *const g_from = (const char *)p.g.ptr + (w.n * p.g.sn + w.head * p.g.sh) * (p.g.dtype == FTC_F32 ? 4 : 2);
    auto request = [&](const Chunk &k) {
        const int all = renewed<NT * HEADS>(threadIdx.x), tid = HEADS == 1 ? all : all % NT;
        if (MODE != kStates) a_tile.fetch(a_from.at(k.base), a_from.row_bytes, width_a, k.valid, tid, flip);
        b_tile.fetch(b_from.at(k.base), b_from.row_bytes, width_a, k.valid, tid, flip);
        c_tile.fetch(c_from.at(k.base), c_from.row_bytes, width_c, k.valid, all, flip);
        if (wave == WAVES - 1) {
            g_next = 0.f;
            const int l = flip ? k.base + k.valid - lane : k.base + lane;  // (reversed: the decay of the position behind)
            if (lane < k.valid && l < w.len)
                g_next = load_as_f32(g_from, p.g.dtype, l * p.g.sl);
        }
    };
    // p's of this chunk, which are wanted in the middle of it
    auto request_p = [&](const Chunk &k) {
        const int tid = renewed<NT * HEADS>(threadIdx.x);
        const int col = mine + 4 * ((tid & 63) >> 4);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int row = 16 * t + (tid & 15);
            const uint32_t off = (uint32_t)(flip ? k.valid - 1 - row : row) * p_from.row_bytes;
            const bool in = row < k.valid && col < width_c;
            if constexpr (VEC) {
                const __amdgpu_buffer_rsrc_t rs = p_from.buffer(k.base);
                const uint32_t from = in ? off + (uint32_t)(col * kB) : kOutside;
                if constexpr (kNarrow) p_own[t] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, from, 0, 0));
                else p_own[t] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, from, 0, 0));
            } else {
                u32x4 x[1] = {u32x4{0u, 0u, 0u, 0u}};
                if (in) {
                    const char *const at = p_from.at(k.base) + off;
                    const int by = max(0, col + 4 - width_c);
                    if (by == 0) {
                        if constexpr (kNarrow) {
                            const Any<2> y = *(const Any<2> *)(at + col * kB);
                            x[0][0] = y.x, x[0][1] = y.y;
                        } else {
                            x[0] = *(const Any<4> *)(at + col * kB);
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < 3; r++)
                            if (col + r < width_c) {
                                if constexpr (kNarrow) x[0][r / 2] |= (uint32_t)((const uint16_t *)at)[col + r] << (16 * (r % 2));
                                else x[0][r] = ((const uint32_t *)at)[col + r];
                            }
                    }
                }
                if constexpr (kNarrow) p_own[t] = u32x2{x[0][0], x[0][1]};
                else p_own[t] = x[0];
            }
        }
    };
    double total = 0.0;  // (the last wavefront's: of the segment's log decays)
    auto factors = [&](float *to) {
        // the sums of log decays in 64 bits: their differences are exponents.  (-1000 stands for everything below: exp of it
        // is zero, and sums of it stay finite.)
        double g = g_next < -1000.f ? -1000.0 : (double)g_next;
        g = sums_so_far(g);
        const double all = of_last_lane(g);
        if (MODE == kStates) total += all;
        g *= 1.4426950408889634;
        const double left = all * 1.4426950408889634 - g;
        const float high = (float)g, low = (float)(g - (double)high), high_left = (float)left;
        to[kHigh * kRows + lane] = high, to[kLow * kRows + lane] = low;
        to[kRise * kRows + lane] = task.inter * power(high, low);
        to[kFall * kRows + lane] = task.write * power(high_left, (float)(left - (double)high_left));
    };

    // ---- the state: rows 16 t + 4 q + r, column mine + c ----
    f32x4 S[ET];
    auto each = [&](auto &&f) {  // f(t, r, row and column of the state)
#pragma unroll
        for (int t = 0; t < ET; t++) {
            const int row = 16 * t + 4 * renewed<4>(q), col = renewed<COLS>(mine + c);  // (a tile's addresses at a time)
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (row + r < width_a && col < width_c) f(t, r, row + r, col);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto clear_state = [&]() {
#pragma unroll
        for (int t = 0; t < ET; t++) S[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    // a user's state: (E, M), rows apart
    auto place = [&](int row, int col, int64_t stride) { return task.transposed ? col * stride + row : row * stride + col; };
    auto of_state = [&](const State &s) { return s.ptr + w.n * s.sn + w.head * s.sh + (int64_t)w.slice * p.width; };
    // a border's: columns of M one after the other, each of slot_rows values along E (zeros behind the last)
    auto slot_quad = [&](int t, const float *slot) { return slot + (mine + c) * p.slot_rows + 16 * t + 4 * q; };
    auto in_slot = [&](int t) { return mine + c < width_c && 16 * t + 4 * q < p.slot_rows; };
    auto load_slot = [&](const float *slot) {
        clear_state();
        if (task.transposed) {
            each([&](int t, int r, int row, int col) { S[t][r] = slot[row * p.slot_rows + col]; });
        } else {
#pragma unroll
            for (int t = 0; t < ET; t++)
                if (in_slot(t)) S[t] = *(const f32x4a *)slot_quad(t, slot);
        }
    };
    auto store_slot = [&](float *slot) {  // (of scans that are not transposed)
#pragma unroll
        for (int t = 0; t < ET; t++)
            if (in_slot(t)) *(f32x4a *)slot_quad(t, slot) = S[t];
    };
    auto decay_of = [&](int l) {  // of one position, 1 past the end
        return l < w.len ? expf(load_as_f32(g_from, p.g.dtype, l * p.g.sl)) : 1.f;
    };
    auto anchor = [&](int border, float dot, int l) {  // X at a border, before position l
#pragma unroll
        for (int d = 1; d < 64; d *= 2) dot += __shfl_xor(dot, d);
        if (lane == 0) p.anchors[((int64_t)w.at * (p.segments + 1) + border) * p.shares + wave] = decay_of(l) * dot;
    };
    // the products of the rows of p with the wavefront's columns of O, from the state or altogether
    auto dots = [&](int which_dots, const f32x4 (&O)[4]) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            f32x4 x;
            if constexpr (kNarrow) x = O[t] * widen(p_own[t]);
            else x = O[t] * __builtin_bit_cast(f32x4, p_own[t]);
            float sum = (x[0] + x[1]) + (x[2] + x[3]);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (q == 0) dot_mem[(which_dots * WAVES + wave) * kRows + 16 * t + c] = sum;
        }
    };

    int seg = first_seg, buffer = 0;
    if (chunks_in(seg) > 0) {
        request(chunk_at(seg, 0));
        if (wave == WAVES - 1) factors(f_mem[0]);
    }
    for (int turn_of = 0; turn_of < segs; turn_of++, seg++) {
        const int border = flip ? seg + 1 : seg, next_border = flip ? seg : seg + 1;
        const bool starts = flip ? seg == p.segments - 1 : seg == 0, ends = flip ? seg == 0 : seg == p.segments - 1;
        if (turn_of == 0) {
            if (!starts && MODE != kStates) {
                load_slot(slots + border * slot_size);
            } else {
                clear_state();
                if (starts && task.first.ptr) {
                    const float *const from = of_state(task.first);
                    each([&](int t, int r, int row, int col) { S[t][r] = from[place(row, col, task.first.sd)]; });
                }
            }
        }
        if (MODE == kPlain && p.anchors) {
            const float *const across = p.across + ((int64_t)w.at * (p.segments + 1) + border) * slot_size;
            f32x4 dot = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < ET; t++)
                if (in_slot(t)) dot += S[t] * *(const f32x4a *)slot_quad(t, across);
            anchor(border, (dot[0] + dot[1]) + (dot[2] + dot[3]), (int)min((int64_t)border * p.seg_len, (int64_t)p.L));
        }
        const int chunks = chunks_in(seg);
        for (int x = 0; x < chunks; x++) {
            const Chunk k = chunk_at(seg, x);
            const float *const fp = f_mem[buffer];
            __syncthreads();  // (what was staged before has been read)
            {
                const int all = renewed<NT * HEADS>(threadIdx.x), tid = HEADS == 1 ? all : all % NT;
                if (MODE != kStates) a_tile.template store_paired<RB>(ap, tid);
                b_tile.template store<RB>(bp, tid);
                if constexpr (kNarrow) c_tile.template store<RC>(cp, all);
                else c_tile.put((lds_float *)cp, kStrideC, all);
            }
            __syncthreads();
            // the next chunk, in this segment or the next one
            Chunk next{0, 0};
            if (x + 1 < chunks) next = chunk_at(seg, x + 1);
            else if (turn_of + 1 < segs && chunks_in(seg + 1) > 0) next = chunk_at(seg + 1, 0);
            if (MODE != kPartner && next.valid > 0) request(next);
            if (partner) request_p(k);
            renew();

            f32x4 O[4] = {};
            if constexpr (MODE != kStates) {
                // tiles of A on and below the diagonal, and the two above it that share a k-step with one, which are zero
                constexpr int XT = (12 + WAVES - 1) / WAVES;
                auto put_A = [&](int m, const f32x4 &x) {
                    const int id = wave + WAVES * m, ti = id < 1 ? 0 : id < 3 ? 1 : id < 6 ? 2 : 3, tj = id - ti * (ti + 1) / 2;
                    if (id < 12)
                        put_pieces<NP>(Ap + Paired<128>::addr(16 * (id < 10 ? ti : 2 * (id - 10)) + c, 4 * (id < 10 ? tj : 2 * (id - 10) + 1) + q), x);
                };
                f32x4 A[XT];
#pragma unroll
                for (int m = 0; m < XT; m++) {
                    const int id = wave + WAVES * m, ti = id < 1 ? 0 : id < 3 ? 1 : id < 6 ? 2 : 3, tj = id - ti * (ti + 1) / 2;
                    A[m] = f32x4{0.f, 0.f, 0.f, 0.f};
                    if (id >= 10) {
                        if (!kOver) put_A(m, A[m]);
                        continue;
                    }
                    constexpr int kAhead = PIECES == 3 ? 1 : kHeld ? 2 : KE;  // k-steps whose operands are read at a time
#pragma unroll
                    for (int s0 = 0; s0 < KE; s0 += kAhead) {
                        Frag left[kAhead][PIECES], right[kAhead][PIECES];
#pragma unroll
                        for (int s = 0; s < kAhead; s++) {
                            rows_apart<RB>(bp, tj, s0 + s, c, q, left[s]);
                            Paired<RB>::rows_of(ap, ti, s0 + s, c, q, right[s]);
                        }
#pragma unroll
                        for (int s = 0; s < kAhead; s++) A[m] = product(left[s], right[s], A[m]);
                    }
                    settle();
                    const int i = 16 * ti + c, j0 = 16 * tj + 4 * q;
                    const f32x4 high = *(const f32x4a *)(fp + kHigh * kRows + j0), low = *(const f32x4a *)(fp + kLow * kRows + j0);
                    const float high_i = fp[kHigh * kRows + i], low_i = fp[kLow * kRows + i];
#pragma unroll
                    for (int r = 0; r < 4; r++) A[m][r] *= task.intra;
                    if (MODE == kPartner && ti == tj)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (j0 + r == i) diag_mem[i] = A[m][r];
#pragma unroll
                    for (int r = 0; r < 4; r++) A[m][r] *= power((high_i - high[r]) + (low_i - low[r]));
                    if (ti == tj)
#pragma unroll
                        for (int r = 0; r < 4; r++) A[m][r] = j0 + r < i + (MODE != kPartner) ? A[m][r] : 0.f;
                    if (!kOver) put_A(m, A[m]);
                }
                {
                    // operands are read ahead of the products before theirs
                    constexpr int kGroup = PIECES == 1 && !kHeld ? 4 : 2, kSteps = 4 / kGroup;
                    Frag af[2][kGroup][PIECES], sf[NP];
                    auto read = [&](int n, Frag (&to)[kGroup][PIECES]) {
#pragma unroll
                        for (int t = 0; t < kGroup; t++) Paired<RB>::rows_of(ap, n % kSteps * kGroup + t, n / kSteps, c, q, to[t]);
                    };
                    read(0, af[0]);
#pragma unroll
                    for (int n = 0; n < KE * kSteps; n++) {
                        if (n + 1 < KE * kSteps) read(n + 1, af[(n + 1) % 2]);
                        if (n % kSteps == 0) cut(S[2 * (n / kSteps)], S[2 * (n / kSteps) + 1], sf);
#pragma unroll
                        for (int order = 2; order >= 0; order--)
#pragma unroll
                            for (int x = 0; x < NP; x++)
                                if (order - x >= 0 && order - x < PIECES)
#pragma unroll
                                    for (int t = 0; t < kGroup; t++)
                                        O[n % kSteps * kGroup + t] = delta::mfma16(sf[x], af[n % 2][t][order - x], O[n % kSteps * kGroup + t]);
                    }
                }
                renew();
                if constexpr (kOver) {
                    __syncthreads();  // (the rows of a have been read)
#pragma unroll
                    for (int m = 0; m < XT; m++) put_A(m, A[m]);
                }
                __syncthreads();
            }
            renew();
            Frag cf[2][PIECES];
            f32x4 C[4];  // row 16 t + 4 q + r, the lane's column
#pragma unroll
            for (int s = 0; s < 2; s++) {
                if constexpr (kNarrow) {
                    columns_of<RC>(cp, wave, s, c, q, cf[s]);
                    C[2 * s] = widen(u32x2{cf[s][0].w[0], cf[s][0].w[1]}), C[2 * s + 1] = widen(u32x2{cf[s][0].w[2], cf[s][0].w[3]});
                } else {
#pragma unroll
                    for (int t = 2 * s; t < 2 * s + 2; t++)
#pragma unroll
                        for (int r = 0; r < 4; r++) C[t][r] = ((const lds_float *)cp)[(16 * t + 4 * q + r) * kStrideC + mine + c];
                    cut(C[2 * s], C[2 * s + 1], cf[s]);
                }
            }
            if constexpr (MODE != kStates) {
#pragma unroll
                for (int t = 0; t < 4; t++) O[t] *= fp[kRise * kRows + 16 * t + c];
                if constexpr (MODE == kPartner) {
                    settle();
                    if (partner) dots(0, O);
                }
                {
                    // (tile, k-step): 0 0, 1 0, 2 0, 3 0, 2 1, 3 1
                    Frag af[2][NP];
                    Paired<128>::rows_of(Ap, 0, 0, c, q, af[0]);
#pragma unroll
                    for (int n = 0; n < 6; n++) {
                        if (n + 1 < 6) Paired<128>::rows_of(Ap, n + 1 < 4 ? n + 1 : n - 1, n + 1 < 4 ? 0 : 1, c, q, af[(n + 1) % 2]);
                        O[n < 4 ? n : n - 2] = product(cf[n < 4 ? 0 : 1], af[n % 2], O[n < 4 ? n : n - 2]);
                    }
                }
                settle();
                if constexpr (MODE == kPartner) {
                    if (partner) dots(1, O);
                    if (next.valid > 0) request(next);
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const float diag = diag_mem[16 * t + c];
                        f32x4 own;  // c's own row
                        if constexpr (kNarrow) {
                            const u32x2 two = *(const __attribute__((address_space(3))) u32x2a *)(cp + Plane<RC>::addr(16 * t + c, 4 * wave + q));
                            own = widen(two);
                        } else {
                            own = *(const __attribute__((address_space(3))) f32x4a *)((const lds_float *)cp + (16 * t + c) * kStrideC + mine + 4 * q);
                        }
                        O[t] += diag * own;
                    }
                }
                if constexpr (HEADS == 2) {
                    // the other chain's result, where the rows of a were: two tiles in either's
                    auto exchange = [&](int t) {
                        return (__attribute__((address_space(3))) f32x4a *)((lds_char *)mem + (t / 2) * (kA + kRowsA)) + (wave * 2 + t % 2) * 64 + lane;
                    };
                    if (half == 1)
#pragma unroll
                        for (int t = 0; t < 4; t++) *exchange(t) = O[t];
                    __syncthreads();
                    if (half == 0)
#pragma unroll
                        for (int t = 0; t < 4; t++) O[t] += *exchange(t);
                }
                if (half == 0 && task.out.ptr) {
                    renew();
                    const int col = mine + 4 * q;
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const int row = 16 * t + c;
                        const uint32_t off = (uint32_t)(flip ? k.valid - 1 - row : row) * out_to.row_bytes + (uint32_t)(col * bytes);
                        const u32x2 half = {delta::to_bf16(O[t][0], O[t][1]), delta::to_bf16(O[t][2], O[t][3])};
                        if constexpr (VEC) {
                            const __amdgpu_buffer_rsrc_t rs = out_to.buffer(k.base);
                            const uint32_t to = row < k.valid && col < width_c ? off : kOutside;
                            if (narrow) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(mfma::u32x2, half), rs, to, 0, 0);
                            else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(mfma::u32x4, O[t]), rs, to, 0, 0);
                        } else if (row < k.valid && col < width_c) {
                            char *const to = out_to.at(k.base) + off;
                            if (col + 4 <= width_c) {
                                if (narrow) *(Any<2> *)to = Any<2>{half.x, half.y};
                                else *(Any<4> *)to = __builtin_bit_cast(u32x4, O[t]);
                            } else {
#pragma unroll
                                for (int r = 0; r < 3; r++)
                                    if (col + r < width_c) {
                                        if (narrow) ((uint16_t *)to)[r] = (uint16_t)(half[r / 2] >> (16 * (r % 2)));
                                        else ((float *)to)[r] = O[t][r];
                                    }
                            }
                        }
                    }
                }
            }
            // the state behind the chunk
            renew();
            const float last = power(fp[kHigh * kRows + kRows - 1], fp[kLow * kRows + kRows - 1]);
#pragma unroll
            for (int t = 0; t < ET; t++) S[t] *= last;
            {
                constexpr int kGroup = PIECES == 1 && KE == 2 ? 4 : 1, kSteps = ET / kGroup;
                Frag bf[2][kGroup][PIECES], wf[3];
                auto read = [&](int n, Frag (&to)[kGroup][PIECES]) {
#pragma unroll
                    for (int t = 0; t < kGroup; t++) columns_of<RB>(bp, n % kSteps * kGroup + t, n / kSteps, c, q, to[t]);
                };
                read(0, bf[0]);
#pragma unroll
                for (int n = 0; n < 2 * kSteps; n++) {
                    const int s = n / kSteps;
                    if (n + 1 < 2 * kSteps) read(n + 1, bf[(n + 1) % 2]);
                    if (n % kSteps == 0)
                        cut(C[2 * s] * *(const f32x4a *)(fp + kFall * kRows + 32 * s + 4 * q),
                            C[2 * s + 1] * *(const f32x4a *)(fp + kFall * kRows + 32 * s + 16 + 4 * q), wf);
#pragma unroll
                    for (int order = 2; order >= 0; order--)
#pragma unroll
                        for (int x = 0; x < PIECES; x++)
                            if (order - x >= 0 && order - x < 3)
#pragma unroll
                                for (int t = 0; t < kGroup; t++)
                                    S[n % kSteps * kGroup + t] = delta::mfma16(bf[n % 2][t][x], wf[order - x], S[n % kSteps * kGroup + t]);
                }
            }
            settle();
            if (wave == WAVES - 1 && next.valid > 0) factors(f_mem[buffer ^ 1]);
            if (partner) {
                __syncthreads();
                if (lane < k.valid && wave < 2) {  // from the state, and altogether
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < WAVES; i++) sum += dot_mem[(wave * WAVES + i) * kRows + lane];
                    task.dots[((int64_t)wave * (p.N * p.H * p.slices) + w.at) * p.L + k.base + (flip ? k.valid - 1 - lane : lane)] = sum;
                }
            }
            buffer ^= 1;
        }
        // behind the segment
        if (MODE == kStates) {
            store_slot(slots + next_border * slot_size);
            if (wave == WAVES - 1 && lane == 0 && w.slice == 0)
                p.totals[(int64_t)(w.n * p.H + w.head) * p.segments + seg] = total;
            return;
        }
        if (half == 0 && task.out.ptr) {  // positions behind the sequence's end
            int start, end;
            segment(seg, start, end);
            const int stop = (int)min((int64_t)start + p.seg_len, (int64_t)p.L), from = max(start, w.len);
            const int col = threadIdx.x % COLS;  // (of the first chain's threads)
            if (col < width_c)
                for (int l = from + threadIdx.x / COLS; l < stop; l += NT / COLS) {
                    char *const to = out_to.at(l) + col * bytes;
                    if (narrow) *(uint16_t *)to = 0;
                    else *(float *)to = 0.f;
                }
        }
        if (MODE != kPlain) continue;
        if (slots && (p.walk || ends)) store_slot(slots + next_border * slot_size);
        if (ends) {
            if (p.last.ptr) {  // (the gradient of the state that was handed in is behind the first position's decay)
                float *const to = of_state(p.last);
                const float factor = flip ? decay_of(0) : 1.f;
                each([&](int t, int r, int row, int col) { to[place(row, col, p.last.sd)] = factor * S[t][r]; });
            }
            if (p.anchors) {
                float dot = 0.f;
                if (p.across_first.ptr) {
                    const float *const first = of_state(p.across_first);
                    each([&](int t, int r, int row, int col) { dot = fmaf(S[t][r], first[place(row, col, p.across_first.sd)], dot); });
                }
                anchor(0, dot, 0);
            }
        }
    }
}

template <typename T, int KE, int WAVES, int MODE, int HEADS>
void launch_heads(const Args &p, hipStream_t stream) {
    const int64_t count = MODE == kStates ? p.segments - 1 : p.walk ? 1 : p.segments;
    const int64_t units = (int64_t)p.N * p.H * p.slices / HEADS * count;
    const dim3 grid((uint32_t)((units + 7) / 8 * 8 * p.tasks));
    bool vec = true;
    for (int i = 0; i < p.tasks; i++)
        for (const Rows *r : {&p.task[i].a, &p.task[i].b, &p.task[i].c, &p.task[i].p, &p.task[i].out}) vec = vec && (!r->ptr || r->vec);
    if (vec) decay_scan_kernel<T, KE, WAVES, MODE, true, HEADS><<<grid, 64 * WAVES * HEADS, 0, stream>>>(p);
    else decay_scan_kernel<T, KE, WAVES, MODE, false, HEADS><<<grid, 64 * WAVES * HEADS, 0, stream>>>(p);
}
template <typename T, int KE, int WAVES, int MODE>
void launch(const Args &p, hipStream_t stream) {
    if constexpr (MODE == kPartner && Elem<T>::kPieces == 1)
        if (p.pairs) return launch_heads<T, KE, WAVES, MODE, 2>(p, stream);
    launch_heads<T, KE, WAVES, MODE, 1>(p, stream);
}
template <typename T, int MODE>
void choose(const Args &p, int depth, int columns, hipStream_t stream) {
    const bool wide = columns_at_once(columns) == 128;
    if (depth <= 64) wide ? launch<T, 2, 8, MODE>(p, stream) : launch<T, 2, 4, MODE>(p, stream);
    else wide ? launch<T, 4, 8, MODE>(p, stream) : launch<T, 4, 4, MODE>(p, stream);
}

}  // namespace
}  // namespace decay
}  // namespace ftc
