// The gated delta rule's state from chunk to chunk, forward (Z of every position, the state before every chunk and
// after the last) and backward (the gradient of the state, dE = dV).  Formulas and layouts: ftc_delta_kernel.h.
//
// A wavefront owns 16 columns of one chain's state in registers and walks the chunks.  What it multiplies with it reads
// as fragments, each one's next chunk requested as soon as this chunk's is used: where there are few wavefronts straight
// into the registers of the operands, without a barrier; where there are many, two or four wavefronts share them in LDS.  A
// chunk is a chain of dependent products, so what bounds few chains is its latency (1.5 us forward, 2.3 back at
// 64 x 64, 2.3 and 3.3 at 128 x 128); many are bound by what a compute unit gets from its caches.
#include "ftc_delta_kernel.h"

namespace ftc {
namespace delta {
namespace {

// Keeps the requests of a phase where they are written
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

// One factor of a chunk's rows: a float a lane from memory, through LDS to the rows 16 t + 4 q .. of the tiles
struct FactorRow {
    float x;
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, int which, int lane) {
        x = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, 4 * (kRows * which + lane), 0, 0));
    }
    __device__ __forceinline__ void put(lds_float *to, int lane) const { to[lane] = x; }
    __device__ static __forceinline__ f32x4 rows(const lds_float *from, int t, int q) {
        return *(const __attribute__((address_space(3))) f32x4a *)(from + 16 * t + 4 * q);
    }
};
__device__ __forceinline__ void load_tiles(const float *from, f32x4 (&x)[4]) {
#pragma unroll
    for (int t = 0; t < 4; t++) x[t] = *(const f32x4a *)(from + 256 * t);
}
__device__ __forceinline__ void store_tiles(float *to, const f32x4 (&x)[4]) {
#pragma unroll
    for (int t = 0; t < 4; t++) *(f32x4a *)(to + 256 * t) = x[t];
}

// A left operand of N fragments: a wavefront that works alone holds it in registers; W that share it keep it in LDS, and
// each carries every W-th piece of the next chunk's on its way there.
// Up to one wavefront a compute unit they work alone, up to two in pairs, above four together.  Each alone fetches all its
// operands, 34 to 64 KB a chunk, and what a compute unit gets from the L2 beside latency is some 20 bytes a clock: more of them
// wait for each other.  Measured (forward and back, us, alone | pairs | four), bf16, 64 chunks of 128 x 128: 256 wavefronts
// 166, 229 | 187, 270 | 213, 327; 512: 261, 326 | 216, 305 | 243, 355; 768: 322, 464 | 295, 413 | 249, 380; 1024: 400, 561 | 340, 490 | 287, 422.
// fp32, 32 chunks of 64 x 64: 256: 86, 119 | 100, 155 | 109, 187; 512: 150, 193 | 121, 172 | 135, 205; 1024: 263, 386 | 226, 327 | 225, 321.
// (Three pieces of 128 key columns do not fit the registers alone, nor in pairs without spills: always four.)
// Four, 1024 wavefronts of 128 x 128 move 1.2 GB in 290 us and 2.0 in 425: 4.3 and 4.7 TB/s, states and results of fp32 for the most.
template <int W, int N, int PIECES>
struct Left {
    static constexpr bool SHARE = W > 1;
    static constexpr int kCount = N * PIECES, kPer = SHARE ? (kCount + W - 1) / W : 1;
    Frag held[SHARE ? 1 : N][SHARE ? 1 : PIECES];
    u32x4 carried[kPer];
    __device__ __forceinline__ void load(const uint16_t *from, int wave, int lane) {
        if constexpr (SHARE) {
#pragma unroll
            for (int i = 0; i < kPer; i++)
                if (kCount % W == 0 || i + 1 < kPer || wave + W * i < kCount)
                    carried[i] = *(const u32x4a *)(from + (wave + W * i) * 512 + 8 * lane);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) load_frag(from, i, lane, held[i]);
        }
    }
    __device__ __forceinline__ void put(lds_char *to, int wave, int lane) const {
        if constexpr (SHARE)
#pragma unroll
            for (int i = 0; i < kPer; i++)
                if (kCount % W == 0 || i + 1 < kPer || wave + W * i < kCount)
                    *(__attribute__((address_space(3))) u32x4a *)(to + (wave + W * i) * 1024 + 16 * lane) = carried[i];
    }
    __device__ __forceinline__ void get(const lds_char *from, int number, int lane, Frag (&a)[PIECES]) const {
#pragma unroll
        for (int k = 0; k < PIECES; k++) {
            if constexpr (SHARE) {
                const u32x4 x = *(const __attribute__((address_space(3))) u32x4a *)(from + (number * PIECES + k) * 1024 + 16 * lane);
                a[k] = Frag{{x.x, x.y, x.z, x.w}};
            } else {
                a[k] = held[number][k];
            }
        }
    }
};
// What was written to LDS is there for all, and what was read may be overwritten
template <int W>
__device__ __forceinline__ void meet() {
    phase();
    if (W > 1) mfma::wg_barrier();
    phase();
}

// Workgroups go to the eight dies in turn: those of one chain to the same, whose cache they share
__device__ __forceinline__ bool place(const DeltaArgs &p, int groups, int &chain, int &group) {
    const uint32_t die = blockIdx.x % 8u, slot = blockIdx.x / 8u;
    chain = (int)(slot / (uint32_t)groups * 8u + die), group = (int)(slot % (uint32_t)groups);
    return chain < p.N * p.H;
}

// ---- segments ----
// Few chains are walked in segments.  A first launch (MAP) walks all but the last: the first one as it is, the others from
// a state of zeros and, as further columns without rows of their own, from the identity: what they add, and the
// linear map that they are.  The second launch makes its segment's first state of those before it, and walks it.  (In
// reverse the same from the other end.)
template <bool MAP>
__host__ __device__ __forceinline__ int blocks_of(const DeltaArgs &p) {
    return p.col_blocks + (MAP ? (p.E + kCols - 1) / kCols : 0);
}
struct Part {
    int chain, segment, block, first, end;
    bool none, here, map, last;  // here: its tiles are stored; map: columns of the identity; last: of the segments, on the way
};
template <int W, bool MAP, bool BACK>
__device__ __forceinline__ Part part_of(const DeltaArgs &p, int wave) {
    Part a;
    int group;
    const int per = (blocks_of<MAP>(p) + W - 1) / W, count = p.segments > 1 ? p.segments - 1 : 1;
    a.none = !place(p, per * count, a.chain, group);
    const int turn = group / per + (!MAP && p.segments > 1 ? 1 : 0);  // on the way
    const int block0 = (group - group / per * per) * W;
    a.segment = scalar(BACK ? p.segments - 1 - turn : turn), a.block = scalar(block0 + wave);
    a.last = turn == p.segments - 1;
    a.none = a.none || (MAP && turn == 0 && block0 >= p.col_blocks);
    a.here = a.block < p.col_blocks && (!MAP || turn == 0), a.map = MAP && a.block >= p.col_blocks;
    a.first = scalar(a.segment * p.seg_chunks), a.end = scalar((a.segment + 1) * p.seg_chunks);
    return a;
}
// What a segment's first launch leaves: states of col_blocks blocks, then the map, tile by tile as a left operand of mfma4
__device__ __forceinline__ float *segment_of(const DeltaArgs &p, int chain, int segment, int tiles) {
    return p.seg + ((int64_t)chain * p.segments + segment) * blocks_of<true>(p) * tiles * 256;
}
template <int KE, bool MAP, bool BACK>
__device__ __forceinline__ void first_state(const DeltaArgs &p, const Part &a, const Where &w, const StateRef &from, int lane,
                                            f32x4 (&S)[2 * KE]) {
    constexpr int ET = 2 * KE;
    const int c = lane & 15, q = lane >> 4, col = kCols * a.block + c, home = BACK ? p.segments - 1 : 0;
    const bool given = from.ptr && a.segment == home && !a.map;
#pragma unroll
    for (int t = 0; t < ET; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int e = 16 * t + 4 * q + r;
            S[t][r] = given && e < p.E && col < p.M ? from.ptr[w.n * from.stride_n + w.h * from.stride_h + e * from.stride_d + col]
                      : MAP && a.map && e == col - kCols * p.col_blocks && a.segment != home ? 1.f : 0.f;
        }
    if (MAP || p.segments == 1 || a.block >= p.col_blocks) return;
    const float *const start = segment_of(p, w.chain, home, ET) + (a.block * ET * 64 + lane) * 4;
#pragma unroll
    for (int t = 0; t < ET; t++) S[t] = *(const f32x4a *)(start + 256 * t);
    const int keys = (p.E + kCols - 1) / kCols, step = BACK ? -1 : 1;
    for (int g = home + step; g != a.segment; g += step) {
        const float *const there = segment_of(p, w.chain, g, ET);
        const float *const add = there + (a.block * ET * 64 + lane) * 4, *const map = there + (p.col_blocks * ET * 64 + lane) * 4;
        f32x4 N[ET];
#pragma unroll
        for (int t = 0; t < ET; t++) N[t] = *(const f32x4a *)(add + 256 * t);
#pragma unroll
        for (int b = 0; b < ET; b++) {  // (rows of S behind the last key column are zero)
            f32x4 left[ET];
#pragma unroll
            for (int t = 0; t < ET; t++) left[t] = *(const f32x4a *)(map + 256 * (min(b, keys - 1) * ET + t));
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int t = 0; t < ET; t++) N[t] = mfma4(left[t][r], S[b][r], N[t]);
        }
        settle();
#pragma unroll
        for (int t = 0; t < ET; t++) S[t] = N[t];
    }
}
template <int KE, bool MAP, bool BACK>
__device__ __forceinline__ void last_state(const DeltaArgs &p, const Part &a, const Where &w, const StateRef &to, int lane,
                                           const f32x4 (&S)[2 * KE]) {
    constexpr int ET = 2 * KE;
    const int c = lane & 15, q = lane >> 4, col = kCols * a.block + c;
    settle();
    if (MAP) {
        if (a.block >= blocks_of<true>(p)) return;
        float *const there = segment_of(p, w.chain, a.segment, ET) + a.block * ET * 256;
#pragma unroll
        for (int t = 0; t < ET; t++) {
            if (!a.map) *(f32x4a *)(there + 256 * t + 4 * lane) = S[t];
            else  // row 4 q + r, column c of its block: to the row's lane
#pragma unroll
                for (int r = 0; r < 4; r++) there[256 * t + (4 * q + r + 16 * (c / 4)) * 4 + c % 4] = S[t][r];
        }
        return;
    }
    if (!a.last || !to.ptr) return;
#pragma unroll
    for (int t = 0; t < ET; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int e = 16 * t + 4 * q + r;
            if (e < p.E && col < p.M) to.ptr[w.n * to.stride_n + w.h * to.stride_h + e * to.stride_d + col] = S[t][r];
        }
}

// 64 rows of the wavefront's 16 columns, row by row from memory and through LDS to rows 16 t + 4 q + r of column c.
// Only what comes from memory stays in registers: whatever was done to it where it is requested would wait for it.
template <typename T, bool VEC>
struct ColumnTile {
    static constexpr int kBytes = Elem<T>::kBytes, kLoads = kRows * kCols * kBytes / 1024, kAcross = kCols * kBytes / 16;
    static constexpr int kTile = kRows * kCols * kBytes;
    u32x4 r[VEC ? kLoads : 4];
    uint16_t half[VEC || kBytes == 4 ? 1 : 16];

    // VEC: lane's row 64 / kAcross i + lane / kAcross, 16 bytes of it; else its values one by one
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rs, uint32_t row_bytes, int col0, int width, int valid, int lane) {
        if constexpr (VEC) {
            const int col = col0 + lane % kAcross * (16 / kBytes);
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const int row = 64 / kAcross * i + lane / kAcross;
                r[i] = __builtin_amdgcn_raw_buffer_load_b128(
                    rs, row < valid && col < width ? (uint32_t)row * row_bytes + (uint32_t)(col * kBytes) : kOutside, 0, 0);
            }
        } else {
            const int col = col0 + (lane & 15);
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int row = 16 * t + 4 * (lane >> 4) + x;
                    const uint32_t at = row < valid && col < width ? (uint32_t)row * row_bytes + (uint32_t)(col * kBytes) : kOutside;
                    if constexpr (kBytes == 4) r[t][x] = __builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, 0);
                    else half[4 * t + x] = __builtin_amdgcn_raw_buffer_load_b16(rs, at, 0, 0);
                }
        }
    }
    __device__ __forceinline__ void put(lds_char *to, int lane) const {
        if constexpr (VEC)
#pragma unroll
            for (int i = 0; i < kLoads; i++) *(__attribute__((address_space(3))) u32x4a *)(to + 1024 * i + 16 * lane) = r[i];
    }
    __device__ __forceinline__ f32x4 values(const lds_char *from, int t, int c, int q) const {
        f32x4 x;
        if constexpr (!VEC) {
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = __uint_as_float(kBytes == 4 ? r[t][i] : (uint32_t)half[kBytes == 4 ? 0 : 4 * t + i] << 16);
        } else if constexpr (kBytes == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = *(const lds_float *)(from + 64 * (16 * t + 4 * q + i) + 4 * c);
        } else {
            const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (mfma::lds_s16x4 *)(from + 32 * (16 * t + 4 * q + (c >> 2)) + 8 * (c & 3))));
            x[0] = __uint_as_float(w.x << 16), x[1] = __uint_as_float(w.x & 0xffff0000u);
            x[2] = __uint_as_float(w.y << 16), x[3] = __uint_as_float(w.y & 0xffff0000u);
        }
        return x;
    }
    // the way back: values of the tiles to rows in memory (a buffer drops what lies outside)
    __device__ static __forceinline__ void store(__amdgpu_buffer_rsrc_t rs, uint32_t row_bytes, int col0, int width, int valid,
                                                 int lane, const f32x4 (&x)[4], lds_char *through) {
        const int c = lane & 15, q = lane >> 4;
        auto at = [&](int row, int col) {
            return row < valid && col < width ? (uint32_t)row * row_bytes + (uint32_t)(col * kBytes) : kOutside;
        };
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = 16 * t + 4 * q + i;
                const uint16_t half = __builtin_bit_cast(uint16_t, (__bf16)x[t][i]);
                if constexpr (VEC && kBytes == 4) *(lds_float *)(through + 64 * row + 4 * c) = x[t][i];
                else if constexpr (VEC) *(__attribute__((address_space(3))) uint16_t *)(through + 32 * row + 2 * c) = half;
                else if constexpr (kBytes == 4) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[t][i]), rs, at(row, col0 + c), 0, 0);
                else __builtin_amdgcn_raw_buffer_store_b16(half, rs, at(row, col0 + c), 0, 0);
            }
        if constexpr (VEC) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int i = 0; i < kLoads; i++)
                __builtin_amdgcn_raw_buffer_store_b128(*(__attribute__((address_space(3))) u32x4a *)(through + 1024 * i + 16 * lane), rs,
                    at(64 / kAcross * i + lane / kAcross, col0 + lane % kAcross * (16 / kBytes)), 0, 0);
        }
    }
};
// A chunk's factors
__device__ __forceinline__ __amdgpu_buffer_rsrc_t factor_rows(const DeltaArgs &p, int64_t at) {
    const uint64_t from = (uint64_t)(p.factors + at * (kFactors * kRows));
    return __builtin_amdgcn_make_buffer_rsrc(
        (void *)(((uint64_t)(uint32_t)scalar((int)(from >> 32)) << 32) | (uint32_t)scalar((int)(uint32_t)from)), 0,
        4 * kFactors * kRows, mfma::kRsrcFlags);
}

template <typename T, int KE, bool VEC, int W, bool MAP>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(1, 1))) void delta_scan_kernel(DeltaArgs p) {
    constexpr int PIECES = Elem<T>::kPieces, ET = 2 * KE, kKeys = 4 * KE * PIECES * 512;
    constexpr bool SHARE = W > 1;
    const int lane = threadIdx.x & 63, wave = SHARE ? scalar(threadIdx.x >> 6) : 0, c = lane & 15, q = lane >> 4;
    const Part part = part_of<W, MAP, false>(p, wave);
    if (part.none) return;
    const int block = part.block, col = kCols * block + c;
    const bool here = SHARE || MAP ? part.here : true;  // (the others carry operands, and compute with zeros)
    const Where w = where_of(p, part.chain, 0);
    const int first = part.first, last = min(part.end, chunks_of(w.len));  // (of its chunks, past the last)

    f32x4 S[ET];
    first_state<KE, MAP, false>(p, part, w, p.initial, lane, S);

    const uint32_t v_row = (uint32_t)p.v.stride_l * Elem<T>::kBytes;
    using Tile = ColumnTile<T, VEC>;
    __shared__ __align__(16) char v_mem[W][Tile::kTile];
    __shared__ __align__(16) float f_mem[W][2][kRows];
    __shared__ __align__(16) char kr_mem[SHARE ? 2 * kKeys : 16], kc_mem[SHARE ? 2 * kKeys : 16], t_mem[SHARE ? kTFrags * 3 * 1024 : 16];
    lds_char *const vp = (lds_char *)v_mem[wave], *const krp = (lds_char *)kr_mem, *const kcp = (lds_char *)kc_mem, *const tp = (lds_char *)t_mem;
    lds_float *const fp = (lds_float *)f_mem[wave];
    Left<W, 4 * KE, PIECES> kr, kc;
    Left<W, kTFrags, 3> tf;
    Tile V;
    FactorRow in, out;
    float decay;
    auto load_in = [&](int chunk) { kr.load(p.kr + (w.key_at + chunk) * kKeys, wave, lane); };
    auto load_rows = [&](int chunk) {
        V.load(chunk_rows(p.v, w.n, w.h, (int64_t)chunk * kRows, Elem<T>::kBytes), v_row, kCols * block, p.M,
               min(kRows, w.len - chunk * kRows), lane);
        const __amdgpu_buffer_rsrc_t rs = factor_rows(p, w.at + chunk);
        in.load(rs, kReadK, lane), out.load(rs, kWrite, lane);
        decay = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, 4 * (kRows * kRise + kRows - 1), 0, 0));
    };
    auto load_t = [&](int chunk) { tf.load(p.t + (w.at + chunk) * (kTFrags * 3 * 512), wave, lane); };
    auto load_out = [&](int chunk) { kc.load(p.kc + (w.key_at + chunk) * kKeys, wave, lane); };
    if (first < last) {
        load_rows(first), load_in(first), load_t(first), load_out(first);
        if (SHARE) kr.put(krp, wave, lane), load_in(min(first + 1, last - 1));
    }
    for (int chunk = first; chunk < last; chunk++) {
        const int64_t at = (w.at + chunk) * p.col_blocks + block;
        const int next = min(chunk + 1, last - 1);
        V.put(vp, lane), in.put(fp, lane), out.put(fp + kRows, lane);
        const float fade = decay;
        if (SHARE) meet<W>();
        if (here) {
            float *const to = p.s + at * (ET * 256) + 4 * lane;
#pragma unroll
            for (int t = 0; t < ET; t++) *(f32x4a *)(to + 256 * t) = S[t];
        }
        // E = V - diag(rk e^G) K S
        f32x4 P[4] = {}, Z[4] = {}, read[4], write[4], values[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            values[t] = V.values(vp, t, c, q);
            read[t] = FactorRow::rows(fp, t, q), write[t] = FactorRow::rows(fp + kRows, t, q);
        }
        if (!SHARE) phase();
#pragma unroll
        for (int s = 0; s < KE; s++) {
            Frag sf[3], a[4][PIECES];
#pragma unroll
            for (int t = 0; t < 4; t++) kr.get(krp, t * KE + s, lane, a[t]);
            cut(S[2 * s], S[2 * s + 1], sf);
            products<0>(a, sf, P);
        }
#pragma unroll
        for (int t = 0; t < 4; t++) P[t] = values[t] - read[t] * P[t];
        phase();
        tf.put(tp, wave, lane);
        if (SHARE) load_t(next), load_rows(next);
        else load_rows(next), load_in(next);
        meet<W>();
        // Z = T E (tiles above the diagonal are zero)
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag ef[3], a[4][3];
#pragma unroll
            for (int t = 2 * s; t < 4; t++) tf.get(tp, t_number(t, s), lane, a[t]);
            cut(P[2 * s], P[2 * s + 1], ef);
            if (s == 0) products<0>(a, ef, Z);
            else products<2>(a, ef, Z);
        }
        if (SHARE || MAP) settle();
        if (here) store_tiles(p.z + at * (4 * 256) + 4 * lane, Z);
        // S <- e^{G_64} S + K^T diag(rk beta e^{G_64 - G}) Z
#pragma unroll
        for (int t = 0; t < 4; t++) Z[t] *= write[t];
#pragma unroll
        for (int t = 0; t < ET; t++) S[t] *= fade;
        phase();
        kc.put(kcp, wave, lane);
        if (SHARE) load_out(next);
        else load_t(next);
        meet<W>();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag uf[3], a[ET][PIECES];
#pragma unroll
            for (int t = 0; t < ET; t++) kc.get(kcp, 2 * t + s, lane, a[t]);
            cut(Z[2 * s], Z[2 * s + 1], uf);
            products<0>(a, uf, S);
        }
        phase();
        if (SHARE) kr.put(krp, wave, lane), load_in(min(chunk + 2, last - 1));
        else load_out(next);
        phase();
    }
    last_state<KE, MAP, false>(p, part, w, p.final_, lane, S);
}

// The same walk from the last chunk to the first, on the gradient of the state:
//   dU = A^T dO + diag(rk e^{G_64 - G}) K dS,   dE = T^T diag(beta) dU,
//   dS <- e^{G_64} dS + Q^T diag(rq e^G) dO - K^T diag(rk e^G) dE
// and what the chunk's keys write of <state, its gradient>: the sum of beta Z . diag(rk e^{G_64 - G}) K dS.
template <typename T, int KE, bool VEC, int W, bool MAP>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(1, 1))) void delta_scan_back_kernel(DeltaArgs p) {
    constexpr int PIECES = Elem<T>::kPieces, ET = 2 * KE, kKeys = 4 * KE * PIECES * 512;
    constexpr bool SHARE = W > 1;
    const int lane = threadIdx.x & 63, wave = SHARE ? scalar(threadIdx.x >> 6) : 0, c = lane & 15, q = lane >> 4;
    const Part part = part_of<W, MAP, true>(p, wave);
    if (part.none) return;
    const int block = part.block, col = kCols * block + c;
    const bool here = SHARE || MAP ? part.here : true;  // (the others carry operands, and compute with zeros)
    const Where w = where_of(p, part.chain, 0);
    const int first = part.first, last = min(part.end, chunks_of(w.len));  // (of its chunks, past the last)

    f32x4 S[ET];
    first_state<KE, MAP, true>(p, part, w, p.grad_final, lane, S);

    const uint32_t g_row = (uint32_t)p.go.stride_l * Elem<T>::kBytes, gv_row = (uint32_t)p.gv.stride_l * Elem<T>::kBytes;
    // (three pieces of two k-steps held: the columns of q where the rows of k were, requested while T is used)
    constexpr bool kTurns = !SHARE && KE * PIECES > 4;
    using Tile = ColumnTile<T, VEC>;
    __shared__ __align__(16) char g_mem[W][Tile::kTile], through_mem[W][SHARE ? 16 : Tile::kTile];
    __shared__ __align__(16) float f_mem[W][4][kRows];
    // (shared: the rows of k and the columns of q take turns in one place)
    __shared__ __align__(16) char in_mem[SHARE ? 2 * kKeys : 16], kc_mem[SHARE ? 2 * kKeys : 16], t_mem[SHARE ? kTFrags * 3 * 1024 : 16];
    lds_char *const inp = (lds_char *)in_mem, *const kcp = (lds_char *)kc_mem, *const tp = (lds_char *)t_mem;
    lds_char *const gp = (lds_char *)g_mem[wave], *const through = SHARE ? gp : (lds_char *)through_mem[wave];
    lds_float *const fp = (lds_float *)f_mem[wave];
    using Keys = Left<W, 4 * KE, PIECES>;
    Keys kr, own_q, kc;
    Keys &qc = kTurns ? kr : own_q;
    Left<W, kTFrags, 3> tf;
    Tile Gr;
    FactorRow write, beta, read_q, read_k;
    f32x4 Y[4], Z[4];
    float decay;
    auto tiles = [&](int chunk) { return ((w.at + chunk) * p.col_blocks + (SHARE || MAP ? min(block, p.col_blocks - 1) : block)) * (4 * 256) + 4 * lane; };
    auto load_in = [&](int chunk) { kr.load(p.kr + (w.key_at + chunk) * kKeys, wave, lane); };
    auto load_rows = [&](int chunk) {
        const __amdgpu_buffer_rsrc_t rs = factor_rows(p, w.at + chunk);
        write.load(rs, kWriteBack, lane), beta.load(rs, kBetaBack, lane), read_q.load(rs, kReadQ, lane), read_k.load(rs, kReadBack, lane);
        decay = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, 4 * (kRows * kRise + kRows - 1), 0, 0));
        load_tiles(p.de + tiles(chunk), Y);
        load_tiles(p.z + tiles(chunk), Z);
    };
    auto load_t = [&](int chunk) { tf.load(p.tt + (w.at + chunk) * (kTFrags * 3 * 512), wave, lane); };
    auto load_g = [&](int chunk) {
        Gr.load(chunk_rows(p.go, w.n, w.h, (int64_t)chunk * kRows, Elem<T>::kBytes), g_row, kCols * block, p.M,
                min(kRows, w.len - chunk * kRows), lane);
    };
    auto load_q = [&](int chunk) { qc.load(p.qc + (w.key_at + chunk) * kKeys, wave, lane); };
    auto load_out = [&](int chunk) { kc.load(p.kc + (w.key_at + chunk) * kKeys, wave, lane); };
    if (first < last) {
        const int from = last - 1;
        if (!kTurns) load_q(from);
        load_in(from), load_rows(from), load_t(from), load_g(from), load_out(from);
        if (SHARE) kr.put(inp, wave, lane), load_in(max(from - 1, first));
    }
    for (int chunk = last - 1; chunk >= first; chunk--) {
        const int64_t at = (w.at + chunk) * p.col_blocks + block;
        const int next = max(chunk - 1, first);
        write.put(fp, lane), beta.put(fp + kRows, lane);
        read_q.put(fp + 2 * kRows, lane), read_k.put(fp + 3 * kRows, lane);
        const float fade = decay;
        const bool shut = !MAP && __any(beta.x == kLeastBeta);
        if (SHARE) meet<W>();
        if (here) {
            float *const to = p.ds + at * (ET * 256) + 4 * lane;
#pragma unroll
            for (int t = 0; t < ET; t++) *(f32x4a *)(to + 256 * t) = S[t];
        }
        f32x4 P[4] = {}, D[4], G[4], write_rows[4], beta_rows[4];
#pragma unroll
        for (int t = 0; t < 4; t++) write_rows[t] = FactorRow::rows(fp, t, q), beta_rows[t] = FactorRow::rows(fp + kRows, t, q);
        if (!SHARE) phase();
#pragma unroll
        for (int s = 0; s < KE; s++) {
            Frag sf[3], a[4][PIECES];
#pragma unroll
            for (int t = 0; t < 4; t++) kr.get(inp, t * KE + s, lane, a[t]);
            cut(S[2 * s], S[2 * s + 1], sf);
            products<0>(a, sf, P);
        }
        // diag(beta) dU
#pragma unroll
        for (int t = 0; t < 4; t++) {
            P[t] *= write_rows[t];
            D[t] = MAP && part.map ? P[t] : beta_rows[t] * Y[t] + P[t];
        }
        if (SHARE || MAP) settle();
        if (here) {
            f32x4 written = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 4; t++) written += Z[t] * P[t];
            p.written[at * 64 + lane] = (written[0] + written[1]) + (written[2] + written[3]);
        }
#pragma unroll
        for (int t = 0; t < 4; t++) P[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        phase();
        tf.put(tp, wave, lane);
        if (SHARE) load_t(next), load_rows(next);
        else if (kTurns) load_q(chunk), load_rows(next);
        else load_in(next), load_rows(next);
        if (!SHARE) phase();
        Gr.put(gp, lane);
        if (SHARE) meet<W>();
        // dE = T^T diag(beta) dU
        f32x4 read_q_rows[4], read_k_rows[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            G[t] = Gr.values(gp, t, c, q);
            read_q_rows[t] = FactorRow::rows(fp + 2 * kRows, t, q), read_k_rows[t] = FactorRow::rows(fp + 3 * kRows, t, q);
        }
        if (!SHARE) phase();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag df[3], a[4][3];
            f32x4(&head)[2] = *(f32x4(*)[2])&P[0];
#pragma unroll
            for (int t = 0; t < 2 * s + 2; t++) tf.get(tp, tt_number(t, s), lane, a[t]);
            cut(D[2 * s], D[2 * s + 1], df);
            if (s == 0) products<0>(*(Frag(*)[2][3])&a, df, head);
            else products<0>(a, df, P);
        }
        if (SHARE) phase(), qc.put(inp, wave, lane), load_q(next), load_g(next);
        settle();
        if (here) store_tiles(p.de + at * (4 * 256) + 4 * lane, P);
        if (here && p.gv.ptr) {
#pragma unroll
            for (int t = 0; t < 4; t++) D[t] = P[t];
            // rows of dE that are there for dbeta alone (a branch costs the launch of the maps 10 %, the others 6 % without it)
            if (MAP || shut)
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const f32x4 b = FactorRow::rows(fp + kRows, t, q);
#pragma unroll
                    for (int r = 0; r < 4; r++) D[t][r] = b[r] == kLeastBeta ? 0.f : P[t][r];
                }
            Tile::store(chunk_rows(Operand{p.gv.ptr, p.gv.stride_n, p.gv.stride_h, p.gv.stride_l, 0, 0}, w.n, w.h,
                                   (int64_t)chunk * kRows, Elem<T>::kBytes),
                        gv_row, kCols * block, p.M, min(kRows, w.len - chunk * kRows), lane, D, through);
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            G[t] *= read_q_rows[t];
            P[t] *= -read_k_rows[t];
        }
#pragma unroll
        for (int t = 0; t < ET; t++) S[t] *= fade;
        phase();
        if (!SHARE) load_t(next), load_g(next);
        meet<W>();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag of[3], a[ET][PIECES];
#pragma unroll
            for (int t = 0; t < ET; t++) qc.get(inp, 2 * t + s, lane, a[t]);
            cut(G[2 * s], G[2 * s + 1], of);
            products<0>(a, of, S);
        }
        phase();
        kc.put(kcp, wave, lane);
        if (SHARE) load_out(next);
        else if (kTurns) load_in(next);
        else load_q(next);
        meet<W>();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            Frag ef[3], a[ET][PIECES];
#pragma unroll
            for (int t = 0; t < ET; t++) kc.get(kcp, 2 * t + s, lane, a[t]);
            cut(P[2 * s], P[2 * s + 1], ef);
            products<0>(a, ef, S);
        }
        phase();
        if (SHARE) kr.put(inp, wave, lane), load_in(max(chunk - 2, first));
        else load_out(next);
        phase();
    }
    last_state<KE, MAP, true>(p, part, w, p.grad_initial, lane, S);
    // positions past the end of the sequence
    if (!MAP && part.last && p.gv.ptr && col < p.M)
        for (int l = w.len + q; l < p.L; l += 4)
            store_from_f32(p.gv.ptr, p.gv.dtype, w.n * p.gv.stride_n + w.h * p.gv.stride_h + l * p.gv.stride_l + col, 0.f);
}

template <typename T, int KE, bool VEC, int W, bool MAP>
void launch(const DeltaArgs &p, bool back, hipStream_t stream) {
    const int64_t segments = p.segments > 1 ? p.segments - 1 : 1, groups = (blocks_of<MAP>(p) + W - 1) / W * segments;
    const dim3 grid(((uint32_t)p.N * (uint32_t)p.H + 7) / 8 * 8 * (uint32_t)groups);
    if (back) delta_scan_back_kernel<T, KE, VEC, W, MAP><<<grid, 64 * W, 0, stream>>>(p);
    else delta_scan_kernel<T, KE, VEC, W, MAP><<<grid, 64 * W, 0, stream>>>(p);
}
constexpr bool fits_registers(int pieces, int ke) { return pieces * ke <= 6; }
template <typename T, int KE, bool VEC, bool MAP>
void launch(const DeltaArgs &p, bool back, hipStream_t stream) {
    const int shared_by = delta_scan_shared_by(p, Elem<T>::kPieces == 1, MAP);
    if (shared_by == 4) launch<T, KE, VEC, 4, MAP>(p, back, stream);
    else if constexpr (fits_registers(Elem<T>::kPieces, KE))
        shared_by == 2 ? launch<T, KE, VEC, 2, MAP>(p, back, stream) : launch<T, KE, VEC, 1, MAP>(p, back, stream);
}
template <typename T, int KE, bool VEC>
void launch(const DeltaArgs &p, bool back, hipStream_t stream) {
    if (p.segments > 1) launch<T, KE, VEC, true>(p, back, stream);
    launch<T, KE, VEC, false>(p, back, stream);
}
template <typename T, int KE>
void launch(const DeltaArgs &p, bool vec, bool back, hipStream_t stream) {
    vec ? launch<T, KE, true>(p, back, stream) : launch<T, KE, false>(p, back, stream);
}
int dispatch(const DeltaArgs &p, bool bf16, bool vec, bool back, hipStream_t stream) {
    if (p.E <= 64) bf16 ? launch<bf16_t, 2>(p, vec, back, stream) : launch<float, 2>(p, vec, back, stream);
    else bf16 ? launch<bf16_t, 4>(p, vec, back, stream) : launch<float, 4>(p, vec, back, stream);
    return FTC_OK;
}

}  // namespace

int delta_scan_shared_by(const DeltaArgs &p, bool bf16, bool first) {
    const int blocks = first ? blocks_of<true>(p) : blocks_of<false>(p);
    const int64_t waves = (int64_t)p.N * p.H * blocks * (p.segments > 1 ? p.segments - 1 : 1);
    if (!fits_registers(bf16 ? 1 : 3, p.E <= 64 ? 2 : 4) || waves > 512) return 4;
    return waves > 256 && blocks % 2 == 0 ? 2 : 1;
}
int delta_scan(const DeltaArgs &p, bool bf16, hipStream_t stream) { return dispatch(p, bf16, p.vec_v, false, stream); }
int delta_scan_back(const DeltaArgs &p, bool bf16, hipStream_t stream) { return dispatch(p, bf16, p.vec_go && p.vec_gv, true, stream); }

}  // namespace delta
}  // namespace ftc
