// C ABI entry points of decayed linear attention (include/ftc_causal_product.h): argument checking, workspaces and the
// sequence of launches.  The kernels: ftc_decay_{scan_f32,scan_bf16,finish,step}.hip.
#include <algorithm>
#include <cmath>
#include <cstdio>

#include "ftc_decay_kernel.h"

namespace ftc {
namespace decay {
namespace {

// Calls of up to this many positions run position by position.  Measured, us at 4, 8 and 16 positions with states in and out, by position
// and as a chunk: 8 chains of 64 x 64, fp32, 8.0, 12.9, 22.9 and 13.0; 16 of 128 x 128, bf16, 10.4, 17.0, 29.9 and 17.5; 99 of 25 x 33, fp32,
// 6.5, 8.9, 13.6 and 12.5; 1024 of 64 x 64, bf16, 13.9, 20.8, 33.1 and 24.4; 1024 of 128 x 128, bf16, 39, 56, 89 and 46.5.
constexpr int64_t kStepMost = 8;
constexpr int64_t kMostRowStride = 1 << 22;  // elements between positions: a chunk's offsets stay below 2 GiB

constexpr int64_t kMostLanes = 0xffffffff;  // of a launch

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

struct Sizes {
    int64_t N, H, Hk, L, E, M;
    int32_t dtype;
    bool bf16() const { return dtype == FTC_BF16; }
    int64_t slices() const { return (M + kSlice - 1) / kSlice; }
    int64_t width() const { return M < kSlice ? M : kSlice; }
    int64_t chains() const { return N * H * slices(); }
    int64_t group() const { return H * slices() / Hk; }  // chains that read a key head
    int64_t chunks() const { return (L + kRows - 1) / kRows; }
    // Workgroups of the scans that a compute unit holds at a time, by their LDS and registers, and what a chunk takes with so many, us: a
    // part that they share and one of each.  Measured with one, two and three: 64 x 64 bf16 2.9, 3.8, 4.8, fp32 5.7, 9; 128 x 128 bf16 4.1, 8.5,
    // fp32 10.9; 128 x 64 bf16 3.7, 6.3, fp32 9.1.
    bool narrow() const { return E <= 64 && width() <= 64; }
    int64_t held() const { return bf16() ? (narrow() ? 3 : 2) : narrow() ? 2 : 1; }
    double chunk(double workgroups) const {
        const double size = (double)(E * width()) / (kMaxE * kSlice), each = workgroups / 256;
        const double shared = !narrow() ? 0 : bf16() ? 2.1 : 1.9, own = narrow() ? (bf16() ? 0.9 : 3.6) : bf16() ? 1 + 3.2 * size : 5 + 5 * size;
        // (where their number is none of compute units some have one more: half of that counts)
        return shared * std::ceil(each / held()) + own * (std::max(1.0, each) + std::ceil(each)) / 2;
    }
    // The times of launches in n segments side by side, us: a scan's chunks and a start, and where there are several, the states at the
    // borders and their sums.  Measured by the number of segments, the one that this picks first:
    //   forward: 64 chains of 2048 x 128 x 128, bf16  8: 78 (2 116, 4 79, 6 88)       8 of 4096 x 64 x 64, bf16   32: 31 (8 49, 64 38)
    //            128 of 4096 x 128 x 128, bf16        4: 219 (1 285, 2 234, 8 248)    256 of 4096 x 64 x 64, bf16  3: 180 (1 202, 2 189, 4 194)
    //            256 of 1024 x 128 x 128, bf16        1: 79 (2 79, 4 80, walked)      192 of 2048 x 64 x 64, fp32  4: 160 (1 193, 2 176, 8 164)
    //   with its backward: 80 of 1000 x 64 x 64, fp32 6: 174 (2 226, 4 193, 16 216)   16 of 16384 x 64 x 64, bf16 43: 238 (16 280, 32 245, 128 294)
    //            64 of 2048 x 128 x 128, bf16         4: 262 (8 277)                  32 of 1024 x 128 x 128, fp32 8: 186 (1 456, 4 212, 16 244)
    //            128 on 64 of keys, 4096 x 128 x 128, bf16  4: 782 to 800 (5 913, 8 886)
    double scan(int64_t n, int64_t tasks) const {
        const double all = (double)(tasks * chains() * n);
        return (double)((chunks() + n - 1) / n) * chunk(all) + 5 * std::ceil(all / (256.0 * held()));
    }
    double states(int64_t n) const {
        return n == 1 ? 0 : (bf16() ? 0.4 : 0.25) * (double)((chunks() + n - 1) / n) * chunk((double)(chains() * (n - 1))) + 7 + 0.15 * n;
    }
    double forward(int64_t n) const { return scan(n, 1) + states(n); }
    // (a backward has two such scans, and one of two tasks whose chunks take a third longer)
    double time(int64_t n, bool keep) const { return keep ? 2 * forward(n) + 1.3 * scan(n, 2) : forward(n); }
    // the number of the least time: as many as give every compute unit so many, or as few as may be
    int64_t best(bool keep) const {
        const int64_t longest = kLongest / kRows, first = keep ? std::max<int64_t>(1, (chunks() + longest - 1) / longest) : 1;
        int64_t found = first;
        for (int64_t each = 1; each <= 2 * held(); each++) {
            const int64_t most = std::min(chunks(), each * 256 / std::max<int64_t>(1, chains()));
            if (most <= first) continue;
            const int64_t len = (chunks() + most - 1) / most, n = std::max(first, (chunks() + len - 1) / len);
            if (time(n, keep) < time(found, keep)) found = n;
        }
        return found;
    }
    int64_t cut[2] = {};  // the segments' lengths, of calls that keep nothing and of those that do (settle)
    void settle() {
        for (int keep = 0; keep < 2; keep++) cut[keep] = kRows * std::max<int64_t>(1, (chunks() + best(keep) - 1) / best(keep));
    }
    int64_t seg_len(bool keep) const { return cut[keep]; }
    int64_t segments(bool keep) const { return std::max<int64_t>(1, (L + seg_len(keep) - 1) / seg_len(keep)); }
    // whether the forward has a workgroup go through all segments
    bool walks(bool keep) const { return segments(keep) == 1 || forward(1) <= forward(segments(keep)); }
    // floats (multiples of 64)
    int64_t slots(bool keep) const { return up(chains() * (segments(keep) + 1) * up(E, 4) * width(), 64); }
    int64_t totals(bool keep) const { return up(2 * N * H * segments(keep), 64); }
    int64_t forward_bytes(bool keep) const { return keep || !walks(false) ? 4 * (slots(keep) + totals(keep)) : 0; }
    int64_t shares() const { return columns_at_once((int)width()) / 16; }
    int64_t anchors() const { return up(chains() * (segments(true) + 1) * shares(), 64); }
    int64_t dots() const { return up(2 * chains() * L, 64); }
    int64_t sums() const { return up(2 * H * N * segments(true), 64); }
    // Two chains of a key head share a workgroup of the scans that make their queries' and keys' gradients (ftc_decay_scan_kernel.h)
    bool pairs() const { return bf16() && group() % 2 == 0; }
    int64_t shares_of_keys() const { return group() / (pairs() ? 2 : 1); }
    int64_t part() const { return shares_of_keys() > 1 ? up(N * Hk * shares_of_keys() * L * E, 64) : 0; }
    // Whether every launch of a route has fewer than 2^32 lanes (ftc_decay_scan_kernel.h, ftc_decay_finish.hip)
    static int64_t scan_lanes(int64_t units, int64_t columns) { return up(units, 8) * 4 * columns_at_once((int)columns); }
    bool borders_fit(bool keep) const {
        const int64_t n = segments(keep);
        return scan_lanes(chains() * (n - 1), width()) <= kMostLanes && (n <= 2 || chains() * up(up(E, 4) * width() / 4, 256) <= kMostLanes);
    }
    bool forward_fits(bool keep) const {
        return scan_lanes(chains() * (walks(keep) ? 1 : segments(keep)), width()) <= kMostLanes && (walks(keep) || borders_fit(keep));
    }
    bool backward_fits() const {
        const int64_t n = segments(true), heads = pairs() ? 2 : 1;
        return borders_fit(true) && scan_lanes(chains() * n, width()) <= kMostLanes &&
               2 * heads * scan_lanes(chains() / heads * n, E) <= kMostLanes && N * H * n * seg_len(true) <= kMostLanes;
    }
    int64_t backward() const { return 4 * (slots(true) + totals(true) + anchors() + 2 * dots() + sums() + 2 * part()); }
};

int too_many() { return fail(FTC_ERR_UNSUPPORTED, "too many chains, positions and columns for one call"); }
int check_sizes(Sizes &s) {
    if (s.N < 0 || s.H < 0 || s.Hk < 0 || s.L < 0 || s.E < 0 || s.M < 0) return fail(FTC_ERR_INVALID, "negative size");
    if (s.H > 0 && (s.Hk == 0 || s.H % s.Hk != 0))
        return fail(FTC_ERR_INVALID, "the number of value heads (%lld) must be a multiple of the number of key heads (%lld)",
                    (long long)s.H, (long long)s.Hk);
    if (s.E < 1 || s.E > kMaxE || s.M < 1 || s.M > 512)
        return fail(FTC_ERR_UNSUPPORTED, "decayed attention takes key rows of 1 to 128 values and value rows of 1 to "
                    "512, got %lld and %lld", (long long)s.E, (long long)s.M);
    constexpr int64_t kMost = 0xffffff;  // (workgroups of 256, the smallest that own a chain)
    if (s.N > kMost || s.H > kMost || s.L > 0x7fffff00 || s.N * s.H > kMost) return too_many();
    s.settle();
    return FTC_OK;
}
// ... and whether a route's launches have room for them
int check_forward(const Sizes &s, bool keep) {  // (what is kept is for a backward)
    return s.N * s.H == 0 || (s.forward_fits(keep) && (!keep || s.backward_fits())) ? FTC_OK : too_many();
}
int check_steps(int64_t lanes) { return lanes <= kMostLanes ? FTC_OK : too_many(); }
int check_rows(const ftc_tensor4 *t, const char *name, int64_t N, int64_t H, int64_t L, int64_t X, int dtype) {
    if (!t) return fail(FTC_ERR_INVALID, "%s is null", name);
    if (t->dtype != FTC_F32 && t->dtype != FTC_BF16)
        return fail(FTC_ERR_INVALID, "%s has dtype code %d, expected FTC_F32 or FTC_BF16", name, (int)t->dtype);
    if (dtype >= 0 && t->dtype != dtype)
        return fail(FTC_ERR_INVALID, "%s has dtype code %d, expected %d", name, (int)t->dtype, dtype);
    if (t->size[0] != N || t->size[1] != H || t->size[2] != L || t->size[3] != X)
        return fail(FTC_ERR_INVALID, "%s has shape (%lld,%lld,%lld,%lld), expected (%lld,%lld,%lld,%lld)", name,
                    (long long)t->size[0], (long long)t->size[1], (long long)t->size[2], (long long)t->size[3],
                    (long long)N, (long long)H, (long long)L, (long long)X);
    if (N * H * L == 0) return FTC_OK;
    if (!t->ptr) return fail(FTC_ERR_INVALID, "%s has a null data pointer", name);
    if (X > 1 && t->stride[3] != 1)
        return fail(FTC_ERR_INVALID, "%s must be contiguous in its last dimension (stride %lld)", name, (long long)t->stride[3]);
    if (L > 1 && (t->stride[2] < 0 || t->stride[2] > kMostRowStride))
        return fail(FTC_ERR_UNSUPPORTED, "%s has rows %lld elements apart, at most %lld are supported", name,
                    (long long)t->stride[2], (long long)kMostRowStride);
    return FTC_OK;
}
int check_state(const ftc_tensor4 *t, const char *name, const Sizes &s) {
    if (!t) return FTC_OK;
    if (t->dtype != FTC_F32) return fail(FTC_ERR_INVALID, "%s must be FTC_F32", name);
    if (t->size[0] != s.N || t->size[1] != s.H || t->size[2] != s.E || t->size[3] != s.M)
        return fail(FTC_ERR_INVALID, "%s has shape (%lld,%lld,%lld,%lld), expected (%lld,%lld,%lld,%lld)", name,
                    (long long)t->size[0], (long long)t->size[1], (long long)t->size[2], (long long)t->size[3],
                    (long long)s.N, (long long)s.H, (long long)s.E, (long long)s.M);
    if (s.N * s.H == 0) return FTC_OK;
    if (!t->ptr) return fail(FTC_ERR_INVALID, "%s has a null data pointer", name);
    if (s.M > 1 && t->stride[3] != 1) return fail(FTC_ERR_INVALID, "%s must be contiguous in its last dimension", name);
    return FTC_OK;
}
int check_apart(const ftc_tensor4 *from, const char *from_name, const ftc_tensor4 *to, const char *to_name) {
    if (from && to && from->ptr && from->ptr == to->ptr)
        return fail(FTC_ERR_INVALID, "%s must not overlap %s: parts of a sequence run side by side", to_name, from_name);
    return FTC_OK;
}
// Whether two rows of a tensor may share memory: in the order of the strides, each has to pass all that the smaller ones reach
bool overlaps_itself(const ftc_tensor4 *t) {
    int order[] = {0, 1, 2};
    std::sort(order, order + 3, [&](int a, int b) { return t->stride[a] < t->stride[b]; });
    int64_t reach = t->size[3];
    for (int i : order) {
        if (t->size[i] < 2) continue;
        if (t->stride[i] < reach) return true;
        reach += t->stride[i] * (t->size[i] - 1);
    }
    return false;
}

// Rows of a tensor with `heads` heads; cut: its columns are those of the slices
Rows rows_of(const ftc_tensor4 *t, const Sizes &s, int64_t heads, bool cut) {
    if (!t) return Rows{};
    const int bytes = t->dtype == FTC_F32 ? 4 : 2, lot = 16 / bytes;
    Rows r{t->ptr, t->stride[0], t->stride[1], t->stride[2], (int32_t)t->size[3], (int32_t)(s.H * s.slices() / heads),
           cut && s.slices() > 1 ? kSlice : 0, 0, t->dtype};
    r.vec = r.width % lot == 0 && ((uintptr_t)r.ptr & 15) == 0 && r.sn % lot == 0 && r.sh % lot == 0 && r.sl % lot == 0;
    return r;
}
State state(const ftc_tensor4 *t) {
    return t ? State{(float *)t->ptr, t->stride[0], t->stride[1], t->stride[2]} : State{};
}

struct Inputs {
    Sizes s;
    Scalars g;
    bool per_head;
};
int read_inputs(const ftc_tensor4 *q, const ftc_tensor4 *k, const ftc_tensor4 *v, const ftc_tensor4 *g, Inputs *in) {
    if (!q || !v || !g) return fail(FTC_ERR_INVALID, "queries, values or log_decay is null");
    in->s = Sizes{v->size[0], v->size[1], q->size[1], v->size[2], q->size[3], v->size[3], q->dtype};
    Sizes &s = in->s;
    if (int rc = check_sizes(s)) return rc;
    if (int rc = check_rows(q, "queries", s.N, s.Hk, s.L, s.E, -1)) return rc;
    if (int rc = check_rows(k, "keys", s.N, s.Hk, s.L, s.E, q->dtype)) return rc;
    if (int rc = check_rows(v, "values", s.N, s.H, s.L, s.M, q->dtype)) return rc;
    in->per_head = g->size[0] == 1 && g->size[2] == 1 && (s.N != 1 || s.L != 1);
    if (int rc = check_rows(g, "log_decay", in->per_head ? 1 : s.N, s.H, in->per_head ? 1 : s.L, 1, -1)) return rc;
    in->g = Scalars{g->ptr, g->stride[0], g->stride[1], g->stride[2], g->dtype};
    if (in->per_head) in->g.sn = in->g.sl = 0;
    return FTC_OK;
}
Args args_of(const Inputs &in, const int64_t *lengths, bool keep) {
    const Sizes &s = in.s;
    Args a = {};
    a.tasks = 1, a.lengths = lengths, a.g = in.g;
    a.N = (int32_t)s.N, a.H = (int32_t)s.H, a.slices = (int32_t)s.slices(), a.L = (int32_t)s.L,
    a.width = (int32_t)s.width(), a.slot_rows = (int32_t)up(s.E, 4);
    a.segments = (int32_t)s.segments(keep), a.seg_len = (int32_t)s.seg_len(keep);
    return a;
}
void scan(const Args &a, const Sizes &s, int64_t depth, int64_t columns, bool partner, bool states, hipStream_t stream) {
    (s.bf16() ? decay_scan_bf16 : decay_scan_f32)(a, (int)depth, (int)columns, partner, states, stream);
}
int launched(const char *name) {
    note_kernel(name);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FTC_OK : fail(FTC_ERR_HIP, "%s: %s", name, hipGetErrorString(e));
}
// The states at the segments' borders: what each segment writes, then from border to border
void borders(Args a, const Sizes &s, hipStream_t stream) {
    scan(a, s, s.E, s.width(), false, true, stream);
    if (a.segments > 2) decay_borders(a, a.task[0], stream);
}

int64_t bytes_of(int64_t N, int64_t H, int64_t Hk, int64_t L, int64_t E, int64_t M, int32_t dtype, int what) {
    Sizes s{N, H, Hk, L, E, M, dtype};
    if (dtype != FTC_F32 && dtype != FTC_BF16) return fail(FTC_ERR_INVALID, "unknown dtype code %d", (int)dtype);
    if (int rc = check_sizes(s)) return rc;
    if (N * H == 0) return 0;
    if (what == 0 && L > kStepMost)
        if (int rc = check_forward(s, false)) return rc;
    if (what != 0)
        if (int rc = check_forward(s, true)) return rc;
    return what == 2 ? s.backward() : what == 1 ? s.forward_bytes(true) : L <= kStepMost ? 0 : s.forward_bytes(false);
}

}  // namespace
}  // namespace decay
}  // namespace ftc

using namespace ftc;
using namespace ftc::decay;

extern "C" {

int64_t ftc_decayed_attention_workspace_bytes(int64_t N, int64_t H, int64_t Hk, int64_t L, int64_t E, int64_t M, int32_t dtype) {
    return bytes_of(N, H, Hk, L, E, M, dtype, 0);
}
int64_t ftc_decayed_attention_kept_bytes(int64_t N, int64_t H, int64_t Hk, int64_t L, int64_t E, int64_t M, int32_t dtype) {
    return bytes_of(N, H, Hk, L, E, M, dtype, 1);
}
int64_t ftc_decayed_attention_backward_workspace_bytes(int64_t N, int64_t H, int64_t Hk, int64_t L, int64_t E, int64_t M, int32_t dtype) {
    return bytes_of(N, H, Hk, L, E, M, dtype, 2);
}

int ftc_decayed_attention_plan(int64_t N, int64_t H, int64_t Hk, int64_t L, int64_t E, int64_t M, int32_t dtype, int32_t keep, char *text,
                               size_t text_bytes) {
    if (!text || text_bytes == 0) return fail(FTC_ERR_INVALID, "null argument");
    text[0] = 0;
    Sizes s{N, H, Hk, L, E, M, dtype};
    if (dtype != FTC_F32 && dtype != FTC_BF16) return fail(FTC_ERR_INVALID, "unknown dtype code %d", (int)dtype);
    if (int rc = check_sizes(s)) return rc;
    if (N * H == 0) return FTC_OK;
    if (L == 0 || (!keep && L <= kStepMost)) {
        if (int rc = check_steps(decay_step_lanes(N * H, M, M % 4 == 0))) return rc;
        snprintf(text, text_bytes, "steps");
        return FTC_OK;
    }
    if (int rc = check_forward(s, keep)) return rc;
    const int64_t segments = s.segments(keep);
    snprintf(text, text_bytes, "segments %lld of %lld%s, slices %lld", (long long)segments, (long long)s.seg_len(keep),
             segments > 1 && s.walks(keep) ? " one after the other" : "", (long long)s.slices());
    return FTC_OK;
}

int ftc_decayed_attention(const ftc_tensor4 *queries, const ftc_tensor4 *keys, const ftc_tensor4 *values, const ftc_tensor4 *log_decay,
                          const int64_t *lengths, float scale, const ftc_tensor4 *initial_state, const ftc_tensor4 *out,
                          const ftc_tensor4 *final_state, void *kept, size_t kept_bytes, void *workspace, size_t workspace_bytes,
                          void *stream) {
    Inputs in;
    if (int rc = read_inputs(queries, keys, values, log_decay, &in)) return rc;
    const Sizes &s = in.s;
    if (int rc = check_rows(out, "out", s.N, s.H, s.L, s.M, queries->dtype)) return rc;
    if (int rc = check_state(initial_state, "initial_state", s)) return rc;
    if (int rc = check_state(final_state, "final_state", s)) return rc;
    if (int rc = check_apart(initial_state, "initial_state", final_state, "final_state")) return rc;
    if (s.N * s.H == 0 || (s.L == 0 && !final_state)) return FTC_OK;
    hipStream_t const on = (hipStream_t)stream;
    if (s.L == 0 || (!kept && s.L <= kStepMost)) {
        StepArgs p = {as_operand(queries), as_operand(keys), as_operand(values), in.g, lengths, state(initial_state), state(final_state),
                      as_operand_out(out), (int32_t)s.N, (int32_t)s.H, (int32_t)s.Hk, (int32_t)s.L, (int32_t)s.E, (int32_t)s.M, scale};
        if (int rc = check_steps(decay_step_lanes(s.N * s.H, s.M, decay_step_vec(p)))) return rc;
        decay_steps(p, on);
        return launched("decay_step_kernel");
    }
    const bool keep = kept != nullptr;
    if (int rc = check_forward(s, keep)) return rc;
    const int64_t need = s.forward_bytes(keep);
    void *const at = keep ? kept : workspace;
    if (need > 0 && (!at || (int64_t)(keep ? kept_bytes : workspace_bytes) < need))
        return fail(FTC_ERR_WORKSPACE, "ftc_decayed_attention needs %lld bytes", (long long)need);
    if (need > 0 && ((uintptr_t)at & 255)) return fail(FTC_ERR_WORKSPACE, "the workspace must be 256-byte aligned");
    Args a = args_of(in, lengths, keep);
    Task &t = a.task[0];
    t.a = rows_of(queries, s, s.Hk, false), t.b = rows_of(keys, s, s.Hk, false), t.c = rows_of(values, s, s.H, true);
    t.out = rows_of(out, s, s.H, true);
    t.inter = t.intra = scale, t.write = 1.f;
    t.first = state(initial_state), a.last = state(final_state);
    a.walk = s.walks(keep);
    if (need > 0) t.slots = (float *)at, a.totals = (double *)(t.slots + s.slots(keep));
    if (!a.walk) borders(a, s, on);
    scan(a, s, s.E, s.width(), false, false, on);
    return launched("decay_scan_kernel");
}

int ftc_decayed_attention_backward(const ftc_tensor4 *queries, const ftc_tensor4 *keys, const ftc_tensor4 *values,
                                   const ftc_tensor4 *log_decay, const int64_t *lengths, float scale, const ftc_tensor4 *initial_state,
                                   const void *kept, size_t kept_bytes, const ftc_tensor4 *grad_out, const ftc_tensor4 *grad_final_state,
                                   const ftc_tensor4 *grad_queries, const ftc_tensor4 *grad_keys, const ftc_tensor4 *grad_values,
                                   const ftc_tensor4 *grad_log_decay, const ftc_tensor4 *grad_initial_state, void *workspace,
                                   size_t workspace_bytes, void *stream) {
    Inputs in;
    if (int rc = read_inputs(queries, keys, values, log_decay, &in)) return rc;
    const Sizes &s = in.s;
    if (int rc = check_rows(grad_out, "grad_out", s.N, s.H, s.L, s.M, queries->dtype)) return rc;
    if (int rc = check_state(initial_state, "initial_state", s)) return rc;
    if (int rc = check_state(grad_final_state, "grad_final_state", s)) return rc;
    if (int rc = check_state(grad_initial_state, "grad_initial_state", s)) return rc;
    struct {
        const ftc_tensor4 *t;
        const char *name;
        int64_t N, heads, L, width;
        int dtype;
    } const grads[] = {{grad_queries, "grad_queries", s.N, s.Hk, s.L, s.E, queries->dtype},
                       {grad_keys, "grad_keys", s.N, s.Hk, s.L, s.E, queries->dtype},
                       {grad_values, "grad_values", s.N, s.H, s.L, s.M, queries->dtype},
                       {grad_log_decay, "grad_log_decay", in.per_head ? 1 : s.N, s.H, in.per_head ? 1 : s.L, 1, log_decay->dtype}};
    for (const auto &g : grads)
        if (g.t)
            if (int rc = check_rows(g.t, g.name, g.N, g.heads, g.L, g.width, g.dtype)) return rc;
    if (int rc = check_apart(grad_final_state, "grad_final_state", grad_initial_state, "grad_initial_state")) return rc;
    if (int rc = check_apart(initial_state, "initial_state", grad_initial_state, "grad_initial_state")) return rc;
    if (s.N * s.H == 0 || (s.L == 0 && !grad_initial_state)) return FTC_OK;
    if (s.L == 0) return fail(FTC_ERR_INVALID, "a call of no positions has no backward");
    if (int rc = check_forward(s, true)) return rc;
    if (!kept || (int64_t)kept_bytes < s.forward_bytes(true))
        return fail(FTC_ERR_WORKSPACE, "ftc_decayed_attention_backward needs the %lld bytes that the forward kept", (long long)s.forward_bytes(true));
    if (!workspace || (int64_t)workspace_bytes < s.backward())
        return fail(FTC_ERR_WORKSPACE, "ftc_decayed_attention_backward needs %lld bytes of workspace", (long long)s.backward());
    if (((uintptr_t)kept | (uintptr_t)workspace) & 255) return fail(FTC_ERR_WORKSPACE, "the workspace must be 256-byte aligned");

    hipStream_t const on = (hipStream_t)stream;
    float *next = (float *)workspace;
    auto take = [&](int64_t floats) {
        float *const here = next;
        next += floats;
        return here;
    };
    float *const back_slots = take(s.slots(true));
    double *const totals = (double *)take(s.totals(true));
    float *const anchors = take(s.anchors()), *const x = take(s.dots()), *const y = take(s.dots());
    double *const sums = (double *)take(s.sums());
    float *const parts[2] = {take(s.part()), take(s.part())};
    const Rows q = rows_of(queries, s, s.Hk, false), k = rows_of(keys, s, s.Hk, false), v = rows_of(values, s, s.H, true),
               go = rows_of(grad_out, s, s.H, true);
    const bool shared = s.shares_of_keys() > 1;
    const int64_t heads = s.Hk * s.shares_of_keys();
    auto share = [&](const ftc_tensor4 *grad, float *part) {
        if (!grad) return Rows{};
        if (!shared) return rows_of(grad, s, s.Hk, false);
        return Rows{part, heads * s.L * s.E, s.L * s.E, s.E, (int32_t)s.E, s.pairs() ? 2 : 1, 0, s.E % 4 == 0, FTC_F32};
    };

    // dv, the state's gradient and X at the borders
    Args a = args_of(in, lengths, true);
    a.totals = totals;
    Task &t = a.task[0];
    t.a = k, t.b = q, t.c = go, t.out = rows_of(grad_values, s, s.H, true);
    t.inter = 1.f, t.intra = t.write = scale, t.reverse = 1;
    t.first = state(grad_final_state), t.slots = back_slots, a.last = state(grad_initial_state);
    const bool both = grad_queries || grad_keys || grad_log_decay;
    if (a.segments > 1 && (grad_keys || grad_values || grad_log_decay || grad_initial_state)) borders(a, s, on);
    if (grad_values || grad_log_decay || grad_initial_state) {
        if (grad_log_decay) a.anchors = anchors, a.across = (const float *)kept, a.across_first = state(initial_state), a.shares = (int32_t)s.shares();
        scan(a, s, s.E, s.width(), false, false, on);
    }
    if (both) {
        Args b = args_of(in, lengths, true);
        b.tasks = 0, b.pairs = s.pairs();
        if (grad_queries || grad_log_decay) {
            Task &u = b.task[b.tasks++];
            u.a = go, u.b = v, u.c = k, u.out = share(grad_queries, parts[0]);
            if (grad_log_decay) u.p = q, u.dots = x;
            u.inter = u.intra = scale, u.write = 1.f, u.transposed = 1;
            u.first = state(initial_state), u.slots = (float *)kept;
        }
        if (grad_keys || grad_log_decay) {
            Task &u = b.task[b.tasks++];
            u.a = v, u.b = go, u.c = q, u.out = share(grad_keys, parts[1]);
            if (grad_log_decay) u.p = k, u.dots = y;
            u.inter = 1.f, u.intra = u.write = scale, u.reverse = u.transposed = 1;
            u.first = state(grad_final_state), u.slots = back_slots;
        }
        scan(b, s, s.width(), s.E, true, false, on);
    }
    FinishArgs f = {};
    f.lengths = lengths, f.g = in.g;
    f.N = (int32_t)s.N, f.H = (int32_t)s.H, f.Hk = (int32_t)s.Hk, f.slices = (int32_t)s.slices(), f.L = (int32_t)s.L, f.E = (int32_t)s.E;
    f.every = s.pairs() ? 2 : 1;
    f.segments = a.segments, f.seg_len = a.seg_len, f.per_head = in.per_head;
    f.x = x, f.y = y, f.anchors = anchors, f.shares = (int32_t)s.shares(), f.sums = sums;
    if (grad_log_decay) {
        f.gg = Scalars{grad_log_decay->ptr, grad_log_decay->stride[0], grad_log_decay->stride[1], grad_log_decay->stride[2], grad_log_decay->dtype};
        decay_finish(f, on);
    }
    if (shared && (grad_queries || grad_keys)) {
        const ftc_tensor4 *const to[2] = {grad_queries, grad_keys};
        for (int i = 0; i < 2; i++)
            if (to[i]) f.part[i] = parts[i], f.sum[i] = as_operand_out(to[i]);
        decay_gather(f, on);
    }
    return launched("decay_scan_kernel");
}

int ftc_decayed_attention_step(const ftc_tensor4 *queries, const ftc_tensor4 *keys, const ftc_tensor4 *values, const ftc_tensor4 *log_decay,
                               float scale, const ftc_tensor4 *state_in_out, const ftc_tensor4 *out, void *stream) {
    Inputs in;
    if (int rc = read_inputs(queries, keys, values, log_decay, &in)) return rc;
    const Sizes &s = in.s;
    if (int rc = check_rows(out, "out", s.N, s.H, s.L, s.M, queries->dtype)) return rc;
    if (!state_in_out) return fail(FTC_ERR_INVALID, "state is null");
    if (int rc = check_state(state_in_out, "state", s)) return rc;
    if (s.N * s.H == 0 || s.L == 0) return FTC_OK;
    if (overlaps_itself(state_in_out)) return fail(FTC_ERR_INVALID, "state is written and must not overlap itself");
    StepArgs p = {as_operand(queries), as_operand(keys), as_operand(values), in.g, nullptr, state(state_in_out), state(state_in_out),
                  as_operand_out(out), (int32_t)s.N, (int32_t)s.H, (int32_t)s.Hk, (int32_t)s.L, (int32_t)s.E, (int32_t)s.M, scale};
    if (int rc = check_steps(decay_step_lanes(s.N * s.H, s.M, decay_step_vec(p)))) return rc;
    decay_steps(p, (hipStream_t)stream);
    return launched("decay_step_kernel");
}

}  // extern "C"
