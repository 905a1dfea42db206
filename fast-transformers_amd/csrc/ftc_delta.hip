// C ABI entry points of the gated delta rule (include/ftc_causal_product.h): argument checking, workspaces and the
// sequence of launches.  The kernels: ftc_delta_{prepare,scan,outputs,gradients,step}.hip.
#include <algorithm>
#include <cstdio>

#include "ftc_delta_kernel.h"

namespace ftc {
namespace delta {
namespace {

// Calls of up to this many positions run position by position: a chunk's three launches take as long however
// few of its 64 positions there are.  Measured (us, position by position | in chunks; 4, 8, 12 and 16 positions): 8 chains of 64 x 64,
// fp32, 11, 19, 26, 34 | 25; 512: 13, 21, 29, 37 | 48; 4096: 53, 90, 127, 164 | 310; 8 of 128 x 128, bf16, 14, 25, 35, 46 | 30;
// 512: 28, 45, 60, 74 | 77; 4096: 224, 372, 523, 652 | 565.
constexpr int64_t kStepMost = 8;
constexpr int64_t kMostRowStride = 1 << 22;  // elements between positions: a chunk's offsets stay below 2 GiB

struct Sizes {
    int64_t N, H, Hk, L, E, M;
    int32_t dtype;
    int64_t chunks() const { return (L + kRows - 1) / kRows; }
    int64_t col_blocks() const { return (M + kCols - 1) / kCols; }
    int64_t tiles() const { return E <= 64 ? 4 : 8; }
    int64_t pieces() const { return dtype == FTC_F32 ? 3 : 1; }
    int64_t units() const { return N * H * chunks(); }  // chunks of all chains
    // floats (all multiples of 64)
    int64_t factors() const { return units() * kFactors * kRows; }
    int64_t t() const { return units() * kTFrags * 3 * 256; }
    int64_t keys() const { return N * Hk * chunks() * 2 * tiles() * pieces() * 256; }
    int64_t s() const { return units() * col_blocks() * tiles() * 256; }
    int64_t z() const { return units() * col_blocks() * 4 * 256; }
    // Few chains are walked in segments, side by side: first what each makes of its first state (a linear map and what
    // it adds), then the walk itself.  That is twice the products, so it takes room for four, up to two wavefronts a
    // compute unit; and the maps of the segments before take 1.2 us each at 64 key columns, 4.5 at 128, which n segments
    // of chunks / n chunks pay back while n^2 is below the chunks, or half of them (bf16).  Measured (forward and back, us,
    // whole | in segments): 16 chains of 64 x 64, bf16, 12 chunks 25, 34 | 25, 32; 64: 98, 153 | 53, 71 (8); 256: 370, 587 | 172, 256 (8;
    // 4: 225, 330); 32 chains, 64 chunks: 100, 154 | 81, 129 (4); 40: 105, 160 | 109, 173 (3: not done).  128 x 128: 16
    // chains, 16 chunks 44, 59 | 46, 61 (3: not done); 64: 148, 210 | 116, 167 (4); 4 chains, 128 chunks 276, 400 | 124, 162 (8; 11: 157, 207).
    int64_t segments() const {
        const int64_t waves = N * H * col_blocks(), most = waves > 0 ? 512 / waves : 1, gain = tiles() == 4 || dtype == FTC_F32 ? chunks() : chunks() / 2;
        int64_t n = 1;
        while (n < most && (n + 1) * (n + 1) <= gain) n++;
        if (most < 4 || n < 3) return 1;
        return (chunks() + segment_chunks(n) - 1) / segment_chunks(n);
    }
    int64_t segment_chunks(int64_t n) const { return (chunks() + n - 1) / n; }
    int64_t segment_states() const {
        const int64_t n = segments();
        return n == 1 ? 0 : N * H * n * (col_blocks() + (E + kCols - 1) / kCols) * tiles() * 256;
    }
    int64_t dots() const { return units() * col_blocks() * kRows; }
    // T, keys, factors, states, Z, segments; to be kept for the backward also the transpose of T and O
    int64_t forward(bool keep) const { return 4 * (factors() + (keep ? 2 : 1) * (t() + z()) + 2 * keys() + s() + segment_states()); }
    int64_t backward() const { return 4 * (s() + z() + 2 * dots() + units() * kSums + keys() + segment_states()); }
};

int check_sizes(const Sizes &s) {
    if (s.N < 0 || s.H < 0 || s.Hk < 0 || s.L < 0 || s.E < 0 || s.M < 0) return fail(FTC_ERR_INVALID, "negative size");
    if (s.H > 0 && (s.Hk == 0 || s.H % s.Hk != 0))
        return fail(FTC_ERR_INVALID, "the number of value heads (%lld) must be a multiple of the number of key heads (%lld)",
                    (long long)s.H, (long long)s.Hk);
    if (s.E < 1 || s.E > kMaxE || s.M < 1 || s.M > 512)
        return fail(FTC_ERR_UNSUPPORTED, "the gated delta rule takes key rows of 1 to 128 values and value rows of 1 to "
                    "512, got %lld and %lld", (long long)s.E, (long long)s.M);
    // (a launch has fewer than 2^32 lanes: 2^24 workgroups of 256, of one chunk and 64 columns or less)
    constexpr int64_t kMost = 0xffffff;
    const int64_t groups = (s.col_blocks() + 3) / 4;
    if (s.N > kMost || s.H > kMost || s.L > 0x7fffff00 ||
        (s.N * s.H > 0 && (s.N * s.H > kMost || s.N * s.H * groups > kMost / (s.chunks() > 1 ? s.chunks() : 1))))
        return fail(FTC_ERR_UNSUPPORTED, "too many chains, positions and columns for one call");
    return FTC_OK;
}

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
        return fail(FTC_ERR_INVALID, "%s must be contiguous in its last dimension (stride %lld)", name,
                    (long long)t->stride[3]);
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
bool reads_wide(const Operand &o) {
    const int bytes = o.dtype == FTC_F32 ? 4 : 2, lot = 16 / bytes;
    return o.width % lot == 0 && ((uintptr_t)o.ptr & 15) == 0 && o.stride_n % lot == 0 && o.stride_h % lot == 0 &&
           o.stride_l % lot == 0;
}
Scalars scalars(const ftc_tensor4 *t) {
    return t ? Scalars{t->ptr, t->stride[0], t->stride[1], t->stride[2], t->dtype} : Scalars{};
}
StateRef state(const ftc_tensor4 *t) {
    return t ? StateRef{(float *)t->ptr, t->stride[0], t->stride[1], t->stride[2]} : StateRef{};
}
OperandOut rows_out(const ftc_tensor4 *t) { return t ? as_operand_out(t) : OperandOut{}; }

void place_sizes(const Sizes &s, DeltaArgs *p) {
    p->N = (int32_t)s.N, p->H = (int32_t)s.H, p->Hk = (int32_t)s.Hk, p->L = (int32_t)s.L;
    p->E = (int32_t)s.E, p->M = (int32_t)s.M;
    p->chunks = (int32_t)s.chunks(), p->col_blocks = (int32_t)s.col_blocks();
    p->segments = (int32_t)s.segments(), p->seg_chunks = (int32_t)s.segment_chunks(p->segments);
}
// The inputs that both directions have
int read_inputs(const ftc_tensor4 *q, const ftc_tensor4 *k, const ftc_tensor4 *v, const ftc_tensor4 *g, const ftc_tensor4 *b,
                Sizes *s, DeltaArgs *p) {
    if (!q || !v) return fail(FTC_ERR_INVALID, "queries or values is null");
    *s = Sizes{v->size[0], v->size[1], q->size[1], v->size[2], q->size[3], v->size[3], q->dtype};
    if (int rc = check_sizes(*s)) return rc;
    if (int rc = check_rows(q, "queries", s->N, s->Hk, s->L, s->E, -1)) return rc;
    if (int rc = check_rows(k, "keys", s->N, s->Hk, s->L, s->E, q->dtype)) return rc;
    if (int rc = check_rows(v, "values", s->N, s->H, s->L, s->M, q->dtype)) return rc;
    if (int rc = check_rows(g, "log_decay", s->N, s->H, s->L, 1, -1)) return rc;
    if (int rc = check_rows(b, "beta", s->N, s->H, s->L, 1, -1)) return rc;
    p->q = as_operand(q), p->k = as_operand(k), p->v = as_operand(v);
    p->g = scalars(g), p->b = scalars(b);
    place_sizes(*s, p);
    p->vec_q = reads_wide(p->q), p->vec_k = reads_wide(p->k), p->vec_v = reads_wide(p->v);
    return FTC_OK;
}
void place_forward(const Sizes &s, void *at, bool keep, DeltaArgs *p) {
    float *next = (float *)at;
    auto take = [&](int64_t floats) {
        float *const here = next;
        next += floats;
        return here;
    };
    p->factors = take(s.factors()), p->s = take(s.s()), p->z = take(s.z());
    p->t = (uint16_t *)take(s.t()), p->kr = (uint16_t *)take(s.keys()), p->kc = (uint16_t *)take(s.keys());
    p->seg = take(s.segment_states());
    if (keep) p->o = take(s.z()), p->tt = (uint16_t *)take(s.t());
}
int launched(const char *name) {
    note_kernel(name);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FTC_OK : fail(FTC_ERR_HIP, "%s: %s", name, hipGetErrorString(e));
}

}  // namespace
}  // namespace delta
}  // namespace ftc

using namespace ftc;
using namespace ftc::delta;

extern "C" {

static int64_t delta_bytes(int64_t N, int64_t H, int64_t Hk, int64_t L, int64_t E, int64_t M, int32_t dtype, int what) {
    const Sizes s{N, H, Hk, L, E, M, dtype};
    if (dtype != FTC_F32 && dtype != FTC_BF16) return fail(FTC_ERR_INVALID, "unknown dtype code %d", (int)dtype);
    if (int rc = check_sizes(s)) return rc;
    return what == 2 ? s.backward() : s.forward(what == 1);
}
int64_t ftc_gated_delta_rule_workspace_bytes(int64_t N, int64_t H, int64_t Hk, int64_t L, int64_t E, int64_t M, int32_t dtype) {
    const int64_t bytes = delta_bytes(N, H, Hk, L, E, M, dtype, 0);
    return bytes > 0 && L <= kStepMost ? 0 : bytes;
}
int64_t ftc_gated_delta_rule_kept_bytes(int64_t N, int64_t H, int64_t Hk, int64_t L, int64_t E, int64_t M, int32_t dtype) {
    return delta_bytes(N, H, Hk, L, E, M, dtype, 1);
}
int64_t ftc_gated_delta_rule_backward_workspace_bytes(int64_t N, int64_t H, int64_t Hk, int64_t L, int64_t E, int64_t M,
                                                      int32_t dtype) {
    return delta_bytes(N, H, Hk, L, E, M, dtype, 2);
}

int ftc_gated_delta_plan(int64_t N, int64_t H, int64_t Hk, int64_t L, int64_t E, int64_t M, int32_t dtype, int32_t keep, char *text,
                         size_t text_bytes) {
    if (!text || text_bytes == 0) return fail(FTC_ERR_INVALID, "null argument");
    text[0] = 0;
    const Sizes s{N, H, Hk, L, E, M, dtype};
    if (dtype != FTC_F32 && dtype != FTC_BF16) return fail(FTC_ERR_INVALID, "unknown dtype code %d", (int)dtype);
    if (int rc = check_sizes(s)) return rc;
    if (s.N * s.H == 0) return FTC_OK;
    if (s.L == 0 || (!keep && s.L <= kStepMost)) {
        snprintf(text, text_bytes, "steps");
        return FTC_OK;
    }
    DeltaArgs p = {};
    place_sizes(s, &p);
    const bool bf16 = dtype == FTC_BF16;
    if (p.segments == 1)
        snprintf(text, text_bytes, "chunks %d, scan %d", (int)p.chunks, delta_scan_shared_by(p, bf16, false));
    else
        snprintf(text, text_bytes, "chunks %d, segments %d, maps %d, scan %d", (int)p.chunks, (int)p.segments,
                 delta_scan_shared_by(p, bf16, true), delta_scan_shared_by(p, bf16, false));
    return FTC_OK;
}

int ftc_gated_delta_rule(const ftc_tensor4 *queries, const ftc_tensor4 *keys, const ftc_tensor4 *values,
                         const ftc_tensor4 *log_decay, const ftc_tensor4 *beta, const int64_t *lengths, float scale,
                         int32_t normalize, const ftc_tensor4 *initial_state, const ftc_tensor4 *out,
                         const ftc_tensor4 *final_state, void *kept, size_t kept_bytes, void *workspace,
                         size_t workspace_bytes, void *stream) {
    Sizes s;
    DeltaArgs p = {};
    if (int rc = read_inputs(queries, keys, values, log_decay, beta, &s, &p)) return rc;
    if (int rc = check_rows(out, "out", s.N, s.H, s.L, s.M, queries->dtype)) return rc;
    if (int rc = check_state(initial_state, "initial_state", s)) return rc;
    if (int rc = check_state(final_state, "final_state", s)) return rc;
    if (s.N * s.H == 0) return FTC_OK;
    p.out = rows_out(out), p.initial = state(initial_state), p.final_ = state(final_state);
    p.vec_out = reads_wide(as_operand(out));
    p.lengths = lengths, p.scale = scale, p.normalize = normalize != 0;
    if (s.L == 0 && !final_state) return FTC_OK;
    if (!kept && s.L <= kStepMost) {
        delta_steps(p, (hipStream_t)stream);
        return launched("delta_step_kernel");
    }
    if (s.L == 0) {  // the state as it came
        delta_steps(p, (hipStream_t)stream);
        return launched("delta_step_kernel");
    }
    const int64_t need = s.forward(kept != nullptr);
    void *const at = kept ? kept : workspace;
    if (!at || (int64_t)(kept ? kept_bytes : workspace_bytes) < need)
        return fail(FTC_ERR_WORKSPACE, "ftc_gated_delta_rule needs %lld bytes", (long long)need);
    if ((uintptr_t)at & 255) return fail(FTC_ERR_WORKSPACE, "the workspace must be 256-byte aligned");
    place_forward(s, at, kept != nullptr, &p);
    const bool bf16 = queries->dtype == FTC_BF16;
    delta_prepare(p, bf16, (hipStream_t)stream);
    delta_scan(p, bf16, (hipStream_t)stream);
    delta_outputs(p, bf16, (hipStream_t)stream);
    return launched("delta_scan_kernel");
}

int ftc_gated_delta_rule_backward(const ftc_tensor4 *queries, const ftc_tensor4 *keys, const ftc_tensor4 *values,
                                  const ftc_tensor4 *log_decay, const ftc_tensor4 *beta, const int64_t *lengths,
                                  float scale, int32_t normalize, const void *kept, size_t kept_bytes,
                                  const ftc_tensor4 *grad_out, const ftc_tensor4 *grad_final_state,
                                  const ftc_tensor4 *grad_queries, const ftc_tensor4 *grad_keys,
                                  const ftc_tensor4 *grad_values, const ftc_tensor4 *grad_log_decay,
                                  const ftc_tensor4 *grad_beta, const ftc_tensor4 *grad_initial_state, void *workspace,
                                  size_t workspace_bytes, void *stream) {
    Sizes s;
    DeltaArgs p = {};
    if (int rc = read_inputs(queries, keys, values, log_decay, beta, &s, &p)) return rc;
    if (int rc = check_rows(grad_out, "grad_out", s.N, s.H, s.L, s.M, queries->dtype)) return rc;
    if (int rc = check_state(grad_final_state, "grad_final_state", s)) return rc;
    if (int rc = check_state(grad_initial_state, "grad_initial_state", s)) return rc;
    struct {
        const ftc_tensor4 *t;
        const char *name;
        int64_t heads, width;
        int dtype;
    } const grads[] = {{grad_queries, "grad_queries", s.Hk, s.E, queries->dtype}, {grad_keys, "grad_keys", s.Hk, s.E, queries->dtype},
                       {grad_values, "grad_values", s.H, s.M, queries->dtype}, {grad_log_decay, "grad_log_decay", s.H, 1, log_decay->dtype},
                       {grad_beta, "grad_beta", s.H, 1, beta->dtype}};
    for (const auto &g : grads)
        if (g.t)
            if (int rc = check_rows(g.t, g.name, s.N, g.heads, s.L, g.width, g.dtype)) return rc;
    if (s.N * s.H == 0 || (s.L == 0 && !grad_initial_state)) return FTC_OK;
    if (s.L == 0) return fail(FTC_ERR_INVALID, "a call of no positions has no backward");
    if (!kept || (int64_t)kept_bytes < s.forward(true))
        return fail(FTC_ERR_WORKSPACE, "ftc_gated_delta_rule_backward needs the %lld bytes that the forward kept",
                    (long long)s.forward(true));
    if (!workspace || (int64_t)workspace_bytes < s.backward())
        return fail(FTC_ERR_WORKSPACE, "ftc_gated_delta_rule_backward needs %lld bytes of workspace", (long long)s.backward());
    if (((uintptr_t)kept | (uintptr_t)workspace) & 255)
        return fail(FTC_ERR_WORKSPACE, "the workspace must be 256-byte aligned");
    p.lengths = lengths, p.scale = scale, p.normalize = normalize != 0;
    place_forward(s, (void *)kept, true, &p);
    p.ds = (float *)workspace, p.de = p.ds + s.s(), p.dots = p.de + s.z(), p.written = p.dots + s.dots();
    p.sums = p.written + s.dots();
    p.seg = p.sums + s.units() * kSums;
    p.qc = (uint16_t *)(p.seg + s.segment_states());
    p.go = as_operand(grad_out), p.vec_go = reads_wide(p.go);
    p.gq = rows_out(grad_queries), p.gk = rows_out(grad_keys), p.gv = rows_out(grad_values);
    p.vec_gv = !grad_values || reads_wide(as_operand(grad_values));
    p.gg = scalars(grad_log_decay), p.gb = scalars(grad_beta);
    p.grad_final = state(grad_final_state), p.grad_initial = state(grad_initial_state);
    const bool bf16 = queries->dtype == FTC_BF16;
    delta_pull(p, bf16, (hipStream_t)stream);
    delta_scan_back(p, bf16, (hipStream_t)stream);
    if (grad_queries || grad_keys || grad_log_decay || grad_beta) delta_gradients(p, bf16, (hipStream_t)stream);
    return launched("delta_gradients_kernel");
}

int ftc_gated_delta_step(const ftc_tensor4 *queries, const ftc_tensor4 *keys, const ftc_tensor4 *values,
                         const ftc_tensor4 *log_decay, const ftc_tensor4 *beta, float scale, int32_t normalize,
                         const ftc_tensor4 *state_in_out, const ftc_tensor4 *out, void *stream) {
    Sizes s;
    DeltaArgs p = {};
    if (int rc = read_inputs(queries, keys, values, log_decay, beta, &s, &p)) return rc;
    if (int rc = check_rows(out, "out", s.N, s.H, s.L, s.M, queries->dtype)) return rc;
    if (!state_in_out) return fail(FTC_ERR_INVALID, "state is null");
    if (int rc = check_state(state_in_out, "state", s)) return rc;
    if (s.N * s.H == 0 || s.L == 0) return FTC_OK;
    if (overlaps_itself(state_in_out))
        return fail(FTC_ERR_INVALID, "state is written and must not overlap itself");
    p.out = rows_out(out), p.initial = p.final_ = state(state_in_out);
    p.scale = scale, p.normalize = normalize != 0;
    delta_steps(p, (hipStream_t)stream);
    return launched("delta_step_kernel");
}

}  // extern "C"
