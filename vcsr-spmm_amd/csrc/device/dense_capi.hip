// dense_capi.hip - extern "C" entry points of the dense operators: argument
// checks, workspaces and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <string>
#include <vector>

#include "dense.hpp"
#include "entry.hpp"

namespace {

using namespace vcsr::entry;

bool is_wide(int32_t t) { return t == VCSR_F32 || t == VCSR_BF16; }
size_t size_of(int32_t t) { return t == VCSR_F32 ? 4 : t == VCSR_BF16 ? 2 : 1; }

void range(bool ok, const char* what) {
    if (!ok) throw vcsr::Error(VCSR_ERANGE, what);
}

// Rows are launched as a grid dimension; a product's operand tile, at most 256
// rows, is addressed with 31-bit byte offsets.
constexpr int64_t kMaxRows = (int64_t)1 << 31, kOperandLd = (int64_t)1 << 20;
constexpr int64_t kMaxOut = (int64_t)1 << 42;  // values of a result: its tiles are counted in 32 bits

constexpr int64_t kMaxChunks = (int64_t)1 << 24;  // AdamW: 256 threads each, fewer than 2^32 in all

void check_rows(int64_t M) {
    need(M >= 0, "negative M");
    range(M < kMaxRows, "M over 2^31 - 1");
}
// A matrix argument of `cols` columns; resolves a stride of 0.
void check_matrix(const void* p, int64_t& ld, int64_t cols, int32_t type, const char* what,
                  bool optional, int64_t rows) {
    if (!p) {
        need(optional || rows == 0, what);
        if (ld == 0) ld = cols;
        return;
    }
    if (ld == 0) ld = cols;
    need(ld >= cols, what);
    range(ld <= ((int64_t)1 << 40), what);
    need((uintptr_t)p % size_of(type) == 0, what);
}
void check_operand(const void* p, int64_t& ld, int64_t cols, int32_t type, const char* what,
                   bool optional, int64_t rows) {
    check_matrix(p, ld, cols, type, what, optional, rows);
    range(ld <= kOperandLd, what);
}
void check_vector(const void* p, const char* what, bool optional = false) {
    need(p || optional, what);
    need((uintptr_t)p % 4 == 0, what);
}
void check_workspace(const void* p, size_t have, size_t want) {
    if (!want) return;
    need(p && have >= want, "workspace: too small (see the _workspace function)");
    need((uintptr_t)p % 16 == 0, "workspace: not 16-byte aligned");
}

vcsr_rmsnorm_args checked(const vcsr_rmsnorm_args* args) {
    need(args, "null argument");
    vcsr_rmsnorm_args a = *args;
    check_rows(a.M);
    need(a.C >= 1, "C: at least 1");
    need(is_wide(a.x_type), "x_type: VCSR_F32 or VCSR_BF16");
    need(is_wide(a.y_type) || a.y_type == VCSR_FP8, "y_type: VCSR_F32, VCSR_BF16 or VCSR_FP8");
    need(a.eps >= 0.f && std::isfinite(a.eps), "eps: a finite number, at least 0");
    check_matrix(a.x, a.ldx, a.C, a.x_type, "x: pointer, alignment or stride", false, a.M);
    check_matrix(a.residual, a.ldr, a.C, a.x_type, "residual: alignment or stride", true, a.M);
    check_vector(a.weight, "weight: pointer or alignment");
    check_matrix(a.sum, a.ldsum, a.C, a.x_type, "sum: alignment or stride", true, a.M);
    check_matrix(a.y, a.ldy, a.C, a.y_type, "y: pointer, alignment or stride", false, a.M);
    need((a.y_scale != nullptr) == (a.y_type == VCSR_FP8) || a.M == 0,
         "y_scale: given for VCSR_FP8 and only then");
    check_vector(a.y_scale, "y_scale: alignment", true);
    check_vector(a.rstd, "rstd: alignment", true);
    need(a.y != a.x || a.M == 0 || (a.y_type == a.x_type && a.ldy == a.ldx),
         "y over x: of another type or stride");
    need(!a.residual || a.y != a.residual || (a.y_type == a.x_type && a.ldy == a.ldr),
         "y over residual: of another type or stride");
    need(!a.sum || a.sum != a.y, "sum: another matrix than y");
    need(!a.sum || a.sum != a.x || a.ldsum == a.ldx, "sum over x: of another stride");
    need(!a.sum || a.sum != a.residual || a.ldsum == a.ldr, "sum over residual: of another stride");
    return a;
}

vcsr_rmsnorm_grad_args checked_sizes(const vcsr_rmsnorm_grad_args* args) {
    need(args, "null argument");
    vcsr_rmsnorm_grad_args a = *args;
    check_rows(a.M);
    need(a.C >= 1, "C: at least 1");
    need(is_wide(a.x_type), "x_type: VCSR_F32 or VCSR_BF16");
    need(is_wide(a.y_type), "y_type: VCSR_F32 or VCSR_BF16");
    return a;
}
vcsr_rmsnorm_grad_args checked(const vcsr_rmsnorm_grad_args* args) {
    vcsr_rmsnorm_grad_args a = checked_sizes(args);
    check_matrix(a.dy, a.lddy, a.C, a.y_type, "dy: pointer, alignment or stride", false, a.M);
    check_matrix(a.s, a.lds, a.C, a.x_type, "s: pointer, alignment or stride", false, a.M);
    check_vector(a.weight, "weight: pointer or alignment");
    check_vector(a.rstd, "rstd: pointer or alignment", a.M == 0);
    check_matrix(a.dsum, a.lddsum, a.C, a.x_type, "dsum: alignment or stride", true, a.M);
    check_matrix(a.dx, a.lddx, a.C, a.x_type, "dx: pointer, alignment or stride", false, a.M);
    check_vector(a.dweight, "dweight: alignment", true);
    if (a.M > 0) {
        need(a.dx != a.dsum || a.lddx == a.lddsum, "dx over dsum: of another stride");
        need(a.dx != a.s || a.lddx == a.lds, "dx over s: of another stride");
        need(a.dx != a.dy || (a.x_type == a.y_type && a.lddx == a.lddy),
             "dx over dy: of another type or stride");
    }
    check_workspace(a.workspace, a.workspace_bytes, vcsr::rmsnorm_grad_workspace(a));
    return a;
}

void check_act(int32_t act) {
    need(act >= VCSR_ACT_NONE && act <= VCSR_ACT_SILU, "act: one of VCSR_ACT_*");
}

vcsr_linear_args checked_sizes(const vcsr_linear_args* args) {
    need(args, "null argument");
    vcsr_linear_args a = *args;
    check_rows(a.M);
    need(a.N >= 1 && a.K >= 1, "N, K: at least 1");
    need(is_wide(a.x_type) || a.x_type == VCSR_FP8, "x_type: VCSR_F32, VCSR_BF16 or VCSR_FP8");
    need(is_wide(a.y_type), "y_type: VCSR_F32 or VCSR_BF16");
    check_act(a.act);
    range(a.K <= kOperandLd, "K over 2^20");
    range(a.M <= kMaxOut / a.N, "M x N over 2^42");
    if (a.ldx == 0) a.ldx = a.K;
    if (a.ldw == 0) a.ldw = a.K;
    if (a.ldy == 0) a.ldy = a.N;
    return a;
}
vcsr::Gemm gemm_of(const vcsr_linear_args& a) {
    vcsr::Gemm g;
    g.I = a.M;
    g.J = a.N;
    g.R = a.K;
    g.type = a.x_type;
    g.out_type = a.y_type;
    g.act = a.act;
    g.p = a.x;
    g.ldp = a.ldx;
    g.q = a.w;
    g.ldq = a.ldw;
    g.p_scale = a.x_scale;
    g.q_scale = a.w_scale;
    g.bias = a.bias;
    g.residual = a.residual;
    g.ldr = a.ldr;
    g.z = a.z;
    g.ldz = a.ldz;
    g.out = a.y;
    g.ldo = a.ldy;
    g.part = (float*)a.workspace;
    return g;
}
vcsr_linear_args checked(const vcsr_linear_args* args) {
    vcsr_linear_args a = checked_sizes(args);
    check_operand(a.x, a.ldx, a.K, a.x_type, "x: pointer, alignment or stride", false, a.M);
    check_operand(a.w, a.ldw, a.K, a.x_type, "w: pointer, alignment or stride", false, a.M);
    const bool scaled = a.x_type == VCSR_FP8;
    need(a.M == 0 || ((a.x_scale != nullptr) == scaled && (a.w_scale != nullptr) == scaled),
         "x_scale, w_scale: given for VCSR_FP8 and only then");
    check_vector(a.x_scale, "x_scale: alignment", true);
    check_vector(a.w_scale, "w_scale: alignment", true);
    check_vector(a.bias, "bias: alignment", true);
    check_matrix(a.residual, a.ldr, a.N, a.y_type, "residual: alignment or stride", true, a.M);
    check_matrix(a.z, a.ldz, a.N, a.y_type, "z: alignment or stride", true, a.M);
    check_matrix(a.y, a.ldy, a.N, a.y_type, "y: pointer, alignment or stride", false, a.M);
    need(!a.z || a.z != a.y, "z: another matrix than y");
    need(!a.z || a.z != a.residual, "z: another matrix than the residual");
    need(!a.residual || a.residual != a.y || a.ldr == a.ldy, "residual over y: of another stride");
    check_workspace(a.workspace, a.workspace_bytes, vcsr::gemm_workspace(gemm_of(a)));
    return a;
}

// Blocks read x and w while others write y and z.  Asked once there is a device: of
// buffers that no kernel will touch, none is in the way.
void need_apart(const vcsr_linear_args& a) {
    if (a.M == 0) return;
    need(a.y != a.x && a.y != a.w, "y: another matrix than x and w");
    need(!a.z || (a.z != a.x && a.z != a.w), "z: another matrix than x and w");
}

// The gradient's work: dz (unless dy serves as it is), dbias' partial rows,
// and the two products, whose partial sums share what is behind.
struct LinearGrad {
    vcsr_linear_grad_args a;
    bool own_dz = false;  // dz lies in the workspace
    int64_t lddz = 0;
    size_t dz_bytes = 0, bias_bytes = 0, part_bytes = 0;
    vcsr::Gemm dx, dw;
    size_t bytes() const { return dz_bytes + bias_bytes + part_bytes; }
};

size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

LinearGrad grad_of(const vcsr_linear_grad_args* args) {
    need(args, "null argument");
    LinearGrad w;
    vcsr_linear_grad_args& a = w.a;
    a = *args;
    check_rows(a.M);
    need(a.N >= 1 && a.K >= 1, "N, K: at least 1");
    need(is_wide(a.x_type), "x_type: VCSR_F32 or VCSR_BF16");
    need(is_wide(a.y_type), "y_type: VCSR_F32 or VCSR_BF16");
    check_act(a.act);
    need(a.z || a.act == VCSR_ACT_NONE || a.M == 0, "z: needed for an activation");
    auto stride = [](int64_t& ld, int64_t cols) {
        if (ld == 0) ld = cols;
    };
    stride(a.lddy, a.N);
    stride(a.ldz, a.N);
    stride(a.ldx, a.K);
    stride(a.ldw, a.K);
    stride(a.lddx, a.K);
    stride(a.lddw, a.K);
    if (a.M == 0) return w;
    range(a.N <= kOperandLd && a.K <= kOperandLd, "N, K over 2^20");
    range(a.M <= kMaxOut / (a.N > a.K ? a.N : a.K), "M x N or M x K over 2^42");
    const bool products = a.dx || a.dw;
    w.own_dz = products && (a.act != VCSR_ACT_NONE || a.x_type != a.y_type);
    // Rows of dz on 16-byte boundaries.
    w.lddz = w.own_dz ? ((int64_t)a.N + 7) / 8 * 8 : a.lddy;
    if (w.own_dz) w.dz_bytes = round_up((size_t)a.M * (size_t)w.lddz * size_of(a.x_type));
    if (a.dbias)
        w.bias_bytes = round_up((size_t)vcsr::dz_row_blocks(a.M, a.N, a.y_type) * (size_t)a.N * 4);
    char* base = (char*)a.workspace;
    const void* dz = w.own_dz ? (const void*)base : a.dy;
    float* part = (float*)(base + w.dz_bytes + w.bias_bytes);
    vcsr::Gemm& x = w.dx;
    x.type = x.out_type = a.x_type;
    x.I = a.M;
    x.J = a.K;
    x.R = a.N;
    x.p = dz;
    x.ldp = w.lddz;
    x.q = a.w;
    x.ldq = a.ldw;
    x.q_cols = true;
    x.out = a.dx;
    x.ldo = a.lddx;
    x.part = part;
    vcsr::Gemm& g = w.dw;
    g.type = g.out_type = a.x_type;
    g.I = a.N;
    g.J = a.K;
    g.R = a.M;
    g.p = dz;
    g.ldp = w.lddz;
    g.p_cols = true;
    g.q = a.x;
    g.ldq = a.ldx;
    g.q_cols = true;
    g.out = a.dw;
    g.ldo = a.lddw;
    g.part = part;
    if (a.dx && a.dw)
        w.part_bytes = vcsr::gemm_pair_workspace(g, x);
    else if (a.dx || a.dw)
        w.part_bytes = vcsr::gemm_workspace(a.dx ? x : g);
    return w;
}

LinearGrad checked(const vcsr_linear_grad_args* args) {
    LinearGrad w = grad_of(args);
    vcsr_linear_grad_args& a = w.a;
    check_operand(a.dy, a.lddy, a.N, a.y_type, "dy: pointer, alignment or stride", false, a.M);
    check_matrix(a.z, a.ldz, a.N, a.y_type, "z: pointer, alignment or stride",
                 a.act == VCSR_ACT_NONE, a.M);
    check_operand(a.x, a.ldx, a.K, a.x_type, "x: pointer, alignment or stride", !a.dw, a.M);
    check_operand(a.w, a.ldw, a.K, a.x_type, "w: pointer, alignment or stride", !a.dx, a.M);
    check_matrix(a.dx, a.lddx, a.K, a.x_type, "dx: alignment or stride", true, a.M);
    check_matrix(a.dw, a.lddw, a.K, a.x_type, "dw: alignment or stride", true, a.M);
    check_vector(a.dbias, "dbias: alignment", true);
    if (a.M > 0 && a.dx) {
        need(w.own_dz || a.dx != a.dy, "dx: over dy, which its product reads");
        need(a.dx != a.w, "dx: over w, which its product reads");
        need(a.dx != a.x || !a.dw, "dx: over x, which dw's product reads");
        need(a.dx != a.dw, "dx: another matrix than dw");
    }
    if (a.M > 0 && a.dw) {
        need(w.own_dz || a.dw != a.dy, "dw: over dy, which its product reads");
        need(a.dw != a.x, "dw: over x, which its product reads");
        need(a.dw != a.w || !a.dx, "dw: over w, which dx's product reads");
    }
    check_workspace(a.workspace, a.workspace_bytes, w.bytes());
    return w;
}

hipError_t run_grad(const LinearGrad& w, hipStream_t st) {
    const vcsr_linear_grad_args& a = w.a;
    hipError_t e = hipSuccess;
    if (a.M == 0) {
        const int64_t size = (int64_t)size_of(a.x_type);
        if (a.dw) e = vcsr::launch_zero(a.dw, a.lddw * size, a.N, a.K * size, st);
        if (e == hipSuccess && a.dbias) {
            const int64_t bytes = (int64_t)a.N * 4;
            e = vcsr::launch_zero(a.dbias, bytes, 1, bytes, st);
        }
        return e;
    }
    char* base = (char*)a.workspace;
    // A single block of rows writes dbias itself.
    const int32_t row_blocks = vcsr::dz_row_blocks(a.M, a.N, a.y_type);
    float* const bias_part =
        !a.dbias ? nullptr : row_blocks == 1 ? a.dbias : (float*)(base + w.dz_bytes);
    vcsr::RowSum bias;
    if (a.dbias && row_blocks > 1) bias = vcsr::RowSum{bias_part, a.dbias, row_blocks, a.N};
    if (w.own_dz || bias_part)
        e = vcsr::launch_dz(a, w.own_dz ? base : nullptr, w.lddz, bias_part, st);
    if (e == hipSuccess && a.dx && a.dw) return vcsr::launch_gemm_pair(w.dw, w.dx, bias, st);
    if (e == hipSuccess && bias.P > 0)
        e = vcsr::launch_sum_rows(bias.part, bias.P, bias.C, bias.C, bias.out, st);
    if (e != hipSuccess || (!a.dx && !a.dw)) return e;
    return vcsr::launch_gemm(a.dx ? w.dx : w.dw, st);
}

}  // namespace

struct vcsr_adamw {
    int device = -1;
    vcsr_adamw_tensor* tensors = nullptr;  // on the device
    int2* chunks = nullptr;                // {tensor, chunk of it}
    int32_t n_chunks = 0;
    ~vcsr_adamw() {
        if (tensors) (void)hipFree(tensors);
        if (chunks) (void)hipFree(chunks);
    }
};

extern "C" {

int vcsr_rmsnorm(const vcsr_rmsnorm_args* args, void* stream, float* ms) {
    return guarded([&] {
        const vcsr_rmsnorm_args a = checked(args);
        need_device();
        hipStream_t st = (hipStream_t)stream;
        run_timed(st, ms, [&] { return vcsr::launch_rmsnorm(a, st); });
    });
}

int vcsr_rmsnorm_grad_workspace(const vcsr_rmsnorm_grad_args* args, size_t* bytes) {
    return guarded([&] {
        need(bytes, "null argument");
        *bytes = vcsr::rmsnorm_grad_workspace(checked_sizes(args));
    });
}

int vcsr_rmsnorm_grad(const vcsr_rmsnorm_grad_args* args, void* stream, float* ms) {
    return guarded([&] {
        const vcsr_rmsnorm_grad_args a = checked(args);
        need_device();
        hipStream_t st = (hipStream_t)stream;
        run_timed(st, ms, [&] { return vcsr::launch_rmsnorm_grad(a, st); });
    });
}

int vcsr_linear_workspace(const vcsr_linear_args* args, size_t* bytes) {
    return guarded([&] {
        need(bytes, "null argument");
        const vcsr_linear_args a = checked_sizes(args);
        *bytes = a.M > 0 ? vcsr::gemm_workspace(gemm_of(a)) : 0;
    });
}

int vcsr_linear(const vcsr_linear_args* args, void* stream, float* ms) {
    return guarded([&] {
        const vcsr_linear_args a = checked(args);
        need_device();
        need_apart(a);
        hipStream_t st = (hipStream_t)stream;
        const vcsr::Gemm g = gemm_of(a);
        run_timed(st, ms, [&] { return vcsr::launch_gemm(g, st); });
    });
}

int vcsr_linear_grad_workspace(const vcsr_linear_grad_args* args, size_t* bytes) {
    return guarded([&] {
        need(bytes, "null argument");
        *bytes = grad_of(args).bytes();
    });
}

int vcsr_linear_grad(const vcsr_linear_grad_args* args, void* stream, float* ms) {
    return guarded([&] {
        const LinearGrad w = checked(args);
        need_device();
        hipStream_t st = (hipStream_t)stream;
        run_timed(st, ms, [&] { return run_grad(w, st); });
    });
}

int vcsr_adamw_create(const vcsr_adamw_tensor* tensors, int32_t count, void* stream,
                      vcsr_adamw** out) {
    return guarded([&] {
        need(out, "null argument");
        *out = nullptr;
        need(count >= 0 && (tensors || count == 0), "tensors: null or a negative count");
        std::vector<vcsr_adamw_tensor> list(tensors, tensors + count);
        std::vector<int2> chunks;
        for (int32_t i = 0; i < count; ++i) {
            const vcsr_adamw_tensor& t = list[i];
            const std::string who = "tensor " + std::to_string(i) + ": ";
            auto must = [&](bool ok, const char* what) { need(ok, (who + what).c_str()); };
            must(t.n >= 0, "negative n");
            range(t.n < kMaxChunks * vcsr::kAdamwChunk, (who + "n of 2^35 or more").c_str());
            must(is_wide(t.grad_type), "grad_type: VCSR_F32 or VCSR_BF16");
            must(t.state_type == VCSR_F32 || t.state_type == VCSR_FP8,
                 "state_type: VCSR_F32 or VCSR_FP8");
            must(std::isfinite(t.weight_decay), "weight_decay: not finite");
            if (t.n == 0) continue;
            const bool f8 = t.state_type == VCSR_FP8;
            must(t.param && t.grad && t.m && t.v, "param, grad, m or v: null");
            must(!f8 || (t.m_scale && t.v_scale), "m_scale, v_scale: needed for VCSR_FP8");
            must(((uintptr_t)t.param | (uintptr_t)t.m_scale | (uintptr_t)t.v_scale) % 4 == 0 &&
                     (uintptr_t)t.grad % size_of(t.grad_type) == 0 &&
                     ((uintptr_t)t.m | (uintptr_t)t.v) % size_of(t.state_type) == 0 &&
                     (uintptr_t)t.copy % 2 == 0,
                 "a pointer is not aligned to its type");
            const int64_t n = (t.n + vcsr::kAdamwChunk - 1) / vcsr::kAdamwChunk;
            range((int64_t)chunks.size() + n < kMaxChunks, "tensors: 2^24 or more chunks of 2048");
            for (int64_t k = 0; k < n; ++k) chunks.push_back(make_int2(i, (int)k));
        }
        need_device();
        std::unique_ptr<vcsr_adamw> h(new vcsr_adamw);
        hip_check(hipGetDevice(&h->device), "hipGetDevice");
        hipStream_t st = (hipStream_t)stream;
        h->tensors = upload_array(list, st, "AdamW tensors");
        h->chunks = upload_array(chunks, st, "AdamW chunks");
        h->n_chunks = (int32_t)chunks.size();
        hip_check(hipStreamSynchronize(st), "hipStreamSynchronize");  // the host arrays end here
        *out = h.release();
    });
}

int vcsr_adamw_step(const vcsr_adamw* plan, const vcsr_adamw_hyper* hyper, void* stream,
                    float* ms) {
    return guarded([&] {
        need(plan && hyper, "null argument");
        const vcsr_adamw_hyper& y = *hyper;
        need(std::isfinite(y.lr) && std::isfinite(y.grad_scale), "lr, grad_scale: not finite");
        need(y.beta1 >= 0.0 && y.beta1 < 1.0 && y.beta2 >= 0.0 && y.beta2 < 1.0,
             "beta1, beta2: in [0, 1)");
        need(y.eps >= 0.0 && std::isfinite(y.eps), "eps: a finite number, at least 0");
        need(y.step >= 1, "step: at least 1");
        int device = -1;
        hip_check(hipGetDevice(&device), "hipGetDevice");
        if (device != plan->device)
            throw vcsr::Error(VCSR_ESTATE, "the plan is another device's");
        vcsr::AdamwStep s;
        s.beta1 = (float)y.beta1;
        s.beta2 = (float)y.beta2;
        s.one_minus_beta1 = (float)(1.0 - y.beta1);
        s.one_minus_beta2 = (float)(1.0 - y.beta2);
        s.lr = y.lr;
        s.lr_over_bias1 = (float)(y.lr / (1.0 - std::pow(y.beta1, (double)y.step)));
        s.inv_root_bias2 =
            (float)(1.0 / std::sqrt(1.0 - std::pow(y.beta2, (double)y.step)));
        s.eps = (float)y.eps;
        s.grad_scale = (float)y.grad_scale;
        hipStream_t st = (hipStream_t)stream;
        run_timed(st, ms, [&] {
            return vcsr::launch_adamw(plan->tensors, plan->chunks, plan->n_chunks, s, st);
        });
    });
}

void vcsr_adamw_free(vcsr_adamw* plan) { delete plan; }

// Not part of the interface (no header declares them): the tests run every kernel of
// the products at small sizes through the first, and hold sizes to the kernels that
// they are there for with the others.
void vcsr_test_force_plan(int32_t tile, int32_t stages, int32_t splits, int64_t rows,
                          int32_t together) {
    vcsr::force_plan(vcsr::GemmPlan{tile, stages, splits, 0, rows}, together != 0);
}
// {tile, stages, splits, rows}
int vcsr_test_linear_plan(const vcsr_linear_args* args, int64_t* out) {
    return guarded([&] {
        const vcsr::GemmPlan p = vcsr::gemm_plan(gemm_of(checked_sizes(args)));
        const int64_t v[4] = {p.tile, p.stages, p.splits, p.rows};
        std::copy(v, v + 4, out);
    });
}
// {together, dw's tile and splits, dx's}
int vcsr_test_linear_grad_plan(const vcsr_linear_grad_args* args, int64_t* out) {
    return guarded([&] {
        const LinearGrad w = grad_of(args);
        const vcsr::PairPlan p = vcsr::gemm_pair_plan(w.dw, w.dx);
        const int64_t v[5] = {p.together, p.dw.tile, p.dw.splits, p.dx.tile, p.dx.splits};
        std::copy(v, v + 5, out);
    });
}

}  // extern "C"
