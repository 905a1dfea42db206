// C ABI entry points of the norms around a block (include/ftc_causal_product.h): argument checking, how many workgroups
// take the rows, and the kernel that adds up what they leave for the parameters.  The norms' kernels: ftc_norm_kernel.h.
#include <algorithm>

#include "ftc_norm_kernel.h"

namespace ftc {
namespace norm {
namespace {

// out[row][col] = sum over `count` rows of floats, `stride` apart, in a fixed order: 32 lots of them by 32 columns
struct Fold {
    const float *from;
    void *to;
    int64_t to_stride, from_stride;  // between results; a result's terms start `from_stride` floats apart
    int32_t dtype, results, count, stride;
};
struct FoldArgs {
    Fold fold[kSums + 1];
    int32_t D, folds;
};
__global__ __launch_bounds__(1024) void fold_rows_kernel(FoldArgs p) {
    __shared__ float mem[32][33];
    const int x = threadIdx.x % 32, lot = threadIdx.x / 32, col = blockIdx.x * 32 + x;
    const Fold f = p.fold[blockIdx.y];
    for (int r = blockIdx.z; r < f.results; r += gridDim.z) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        if (col < p.D) {
            const float *const from = f.from + r * f.from_stride + col;
            int i = lot;
            for (; i + 96 < f.count; i += 128)
#pragma unroll
                for (int k = 0; k < 4; k++) sum[k] += from[(int64_t)(i + 32 * k) * f.stride];
            for (; i < f.count; i += 32) sum[0] += from[(int64_t)i * f.stride];
        }
        __syncthreads();
        mem[lot][x] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        __syncthreads();
        // the lots' sums of a column, by the 32 lanes of one of them
        float all = mem[x][lot];
#pragma unroll
        for (int d = 1; d < 32; d *= 2) all += __shfl_xor(all, d);
        const int own = blockIdx.x * 32 + lot;
        if (x == 0 && own < p.D) store_from_f32(f.to, f.dtype, r * f.to_stride + own, all);
    }
}

// ---- host ----
constexpr int64_t kMostWidth = 16384;
constexpr int kLeastNormed = 3;

Plan plan_of(int64_t D, int64_t rows, int64_t segment, bool backward, bool full) {
    Plan q;
    // Lanes to a row, eight values each.  Rows between the sizes leave lanes idle, at worst all but one in sixteen: forward and backward of
    // 2^26 bf16 values with a gate, TB/s: width 16 0.7, 0.8; 64 2.5, 2.6; 96 3.6, 3.5; 128 4.4, 4.2; 136 1.4, 1.5; 256 2.5, 2.5; 384
    // 3.5, 3.4; 512 4.5, 4.2; 520 2.9, 2.4; 768 3.9, 3.4; 1024 4.7, 4.2; 2056 2.6, 1.9; 3000 3.7, 2.6.
    q.lpr = D <= 128 ? 16 : D <= 512 ? 64 : D <= 1024 ? 128 : D <= 2048 ? 256 : D <= 8192 ? 512 : 1024;
    q.teams = q.lpr > 256 ? 1 : 256 / q.lpr;
    // As many as the GPU holds at a time, by their registers (more would wait, and the backward leaves sums with each of
    // them).  Backward of 524288 x 128 with 768 of the lean kernel 143 us, with 512 179; of 40960 x 512 with 512 of the full
    // one 115, with 768 138; forward of either with 1024 95 and 78, with 2048 104 and 82.
    // (forward, teams of 128 lanes and more: rows waiting fill the gaps between a row's loads, sums and stores.  60000 x 1024, bf16, 95 with
    // 4096, with 1024 117; 32768 x 2048 147 and 156; 37735 x 3160 198 with 1536, with 512 242.)
    const int64_t most = q.lpr > 512 ? 256 : !backward ? (q.lpr > 256 ? 1536 : q.lpr > 64 ? 4096 : 1024)
                                              : q.lpr > 256 ? 512 : full ? 512 : 768;
    const int64_t segments = (rows + segment - 1) / segment;
    q.parts = std::min((segment + q.teams - 1) / q.teams, std::max<int64_t>(1, most / segments));
    q.groups = std::min(segments, std::max<int64_t>(1, most / q.parts)) * q.parts;
    return q;
}

int read_rows(const ftc_rows *r, const char *name, bool wanted, Rows *to) {
    *to = Rows{};
    if (!r || !r->ptr) return wanted ? fail(FTC_ERR_INVALID, "%s is null", name) : FTC_OK;
    if (r->dtype != FTC_F32 && r->dtype != FTC_BF16)
        return fail(FTC_ERR_INVALID, "%s has dtype code %d, expected FTC_F32 or FTC_BF16", name, (int)r->dtype);
    *to = Rows{r->ptr, r->stride, r->dtype};
    return FTC_OK;
}
int read_norm(const ftc_norm &n, const char *name, Params *to) {
    if (n.kind < FTC_NORM_NONE || n.kind > FTC_NORM_LAYER) return fail(FTC_ERR_INVALID, "%s has kind %d", name, (int)n.kind);
    for (int32_t d : {n.weight_dtype, n.bias_dtype})
        if (d != FTC_F32 && d != FTC_BF16) return fail(FTC_ERR_INVALID, "%s has dtype code %d", name, (int)d);
    const bool none = n.kind == FTC_NORM_NONE;
    *to = Params{none ? nullptr : n.weight, none ? nullptr : n.bias, n.kind, n.weight_dtype, n.bias_dtype};
    return FTC_OK;
}
int read_call(const ftc_residual_norm_call *c, Args *p) {
    if (!c) return fail(FTC_ERR_INVALID, "the call is null");
    if (c->rows < 0 || c->width < 1 || c->width > kMostWidth || c->rows > 0x7fffffff)
        return fail(c->rows < 0 ? FTC_ERR_INVALID : FTC_ERR_UNSUPPORTED,
                    "rows of 1 to %lld values are supported, and fewer than 2^31 of them", (long long)kMostWidth);
    if (c->activation < FTC_GATE_PLAIN || c->activation > FTC_GATE_SILU)
        return fail(FTC_ERR_INVALID, "the gate's activation has code %d", (int)c->activation);
    p->rows = c->rows, p->D = (int32_t)c->width, p->activation = c->activation, p->scale = c->scale, p->eps = c->eps;
    if (int rc = read_rows(&c->block, "block", c->rows > 0, &p->block)) return rc;
    if (int rc = read_rows(&c->residual, "residual", false, &p->residual)) return rc;
    if (int rc = read_rows(&c->gate, "gate", false, &p->gate)) return rc;
    if (int rc = read_norm(c->after, "the norm after the block", &p->after)) return rc;
    if (int rc = read_norm(c->before, "the norm before the next block", &p->before)) return rc;
    // (a layer norm of two values, or the mean square's of one, has gradients that are all cancellation: eps / r^2 of
    // what is subtracted, which is the rounding of fp32.  One limit for both norms, and for calls without gradients.)
    if (c->width < kLeastNormed && (p->after.kind != FTC_NORM_NONE || p->before.kind != FTC_NORM_NONE))
        return fail(FTC_ERR_UNSUPPORTED, "rows of at least %d values are normalised", kLeastNormed);
    p->gate_rows = p->gate.ptr ? c->gate_rows : 0;
    if (p->gate.ptr && (p->gate_rows < 1 || c->rows % p->gate_rows))
        return fail(FTC_ERR_INVALID, "the gate has %lld rows, which do not divide the block's %lld",
                    (long long)c->gate_rows, (long long)c->rows);
    return FTC_OK;
}
void set_segments(Args *p) {
    p->shared = p->gate.ptr && p->gate_rows < p->rows;
    p->every = p->gate.ptr ? p->rows / p->gate_rows : 1;
    p->segment = p->shared ? p->every : p->rows;
}
Plan backward_plan(const Args &p) { return plan_of(p.D, p.rows, p.segment, true, full(p)); }
int64_t sums_floats(const Args &p, const Plan &q) { return q.groups * kSums * p.D; }
int64_t gate_floats(const Args &p, const Plan &q) { return p.shared ? p.gate_rows * q.parts * p.D : 0; }
int launched(const char *name) {
    note_kernel(name);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FTC_OK : fail(FTC_ERR_HIP, "%s: %s", name, hipGetErrorString(e));
}

}  // namespace
}  // namespace norm
}  // namespace ftc

using namespace ftc;
using namespace ftc::norm;

extern "C" {

int ftc_residual_norm(const ftc_residual_norm_call *call, const ftc_rows *x, const ftc_rows *h, float *stats, void *stream) {
    Args p = {};
    if (int rc = read_call(call, &p)) return rc;
    if (int rc = read_rows(x, "x", p.rows > 0, &p.x)) return rc;
    if (int rc = read_rows(h, "h", p.rows > 0 && p.before.kind != FTC_NORM_NONE, &p.h)) return rc;
    if (p.before.kind == FTC_NORM_NONE && p.h.ptr) return fail(FTC_ERR_INVALID, "h is given without the norm that makes it");
    if (p.rows == 0) return FTC_OK;
    p.stats = stats;
    set_segments(&p);
    const Plan q = plan_of(p.D, p.rows, p.rows, false, false);
    (p.D % kLot ? norm_forward_tail : norm_forward)(p, q, (hipStream_t)stream);
    return launched("residual_norm_kernel");
}

int64_t ftc_residual_norm_backward_workspace_bytes(const ftc_residual_norm_call *call) {
    Args p = {};
    if (int rc = read_call(call, &p)) return rc;
    if (p.rows == 0) return 0;
    set_segments(&p);
    const Plan q = backward_plan(p);
    return 4 * (sums_floats(p, q) + gate_floats(p, q));
}

int ftc_residual_norm_backward(const ftc_residual_norm_call *call, const float *stats, const ftc_rows *grad_x,
                               const ftc_rows *grad_h, const ftc_rows *grad_block, const ftc_rows *grad_residual,
                               const ftc_rows *grad_gate, void *grad_after_weight, void *grad_after_bias,
                               void *grad_before_weight, void *grad_before_bias, void *workspace, size_t workspace_bytes,
                               void *stream) {
    Args p = {};
    if (int rc = read_call(call, &p)) return rc;
    if (int rc = read_rows(grad_x, "grad_x", false, &p.grad_x)) return rc;
    if (int rc = read_rows(grad_h, "grad_h", false, &p.grad_h)) return rc;
    if (int rc = read_rows(grad_block, "grad_block", false, &p.grad_block)) return rc;
    if (int rc = read_rows(grad_residual, "grad_residual", false, &p.grad_residual)) return rc;
    if (int rc = read_rows(grad_gate, "grad_gate", false, &p.grad_gate)) return rc;
    if (p.grad_gate.ptr && !p.gate.ptr) return fail(FTC_ERR_INVALID, "grad_gate is given without a gate");
    if (p.rows == 0) return FTC_OK;
    if (!stats && (p.after.kind != FTC_NORM_NONE || p.before.kind != FTC_NORM_NONE))
        return fail(FTC_ERR_INVALID, "stats is null");
    set_segments(&p);
    const Plan q = backward_plan(p);
    if (!workspace || (int64_t)workspace_bytes < 4 * (sums_floats(p, q) + gate_floats(p, q)))
        return fail(FTC_ERR_WORKSPACE, "ftc_residual_norm_backward needs %lld bytes",
                    (long long)(4 * (sums_floats(p, q) + gate_floats(p, q))));
    if ((uintptr_t)workspace & 255) return fail(FTC_ERR_WORKSPACE, "the workspace must be 256-byte aligned");
    p.stats = const_cast<float *>(stats);
    p.sums = (float *)workspace, p.gate_sums = p.shared ? p.sums + sums_floats(p, q) : nullptr;
    p.parts = (int32_t)q.parts;
    FoldArgs f = {};
    f.D = p.D;
    struct {
        const void *param;
        void *grad;
        int32_t dtype;
    } const params[kSums] = {{p.after.weight, grad_after_weight, p.after.weight_dtype}, {p.after.bias, grad_after_bias, p.after.bias_dtype},
                             {p.before.weight, grad_before_weight, p.before.weight_dtype}, {p.before.bias, grad_before_bias, p.before.bias_dtype}};
    for (int i = 0; i < kSums; i++)
        if (params[i].param && params[i].grad)
            f.fold[f.folds++] = Fold{p.sums + i * p.D, params[i].grad, 0, 0, params[i].dtype, 1, (int32_t)q.groups, kSums * p.D};
    if (!f.folds) p.sums = nullptr;
    int results = 1;
    if (p.shared && p.grad_gate.ptr) {
        results = (int)std::min<int64_t>(p.gate_rows, 4096);
        f.fold[f.folds++] = Fold{p.gate_sums, p.grad_gate.ptr, p.grad_gate.stride, q.parts * p.D, p.grad_gate.dtype,
                                 (int32_t)p.gate_rows, (int32_t)q.parts, p.D};
    } else {
        p.gate_sums = nullptr;
    }
    (p.D % kLot ? norm_backward_tail : norm_backward)(p, q, (hipStream_t)stream);
    if (f.folds)
        fold_rows_kernel<<<dim3((uint32_t)((p.D + 31) / 32), (uint32_t)f.folds, (uint32_t)results), 1024, 0, (hipStream_t)stream>>>(f);
    return launched("residual_norm_backward_kernel");
}

}  // extern "C"
