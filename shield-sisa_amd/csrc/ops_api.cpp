// The C ABI of the operators (include/shv_hip_ops.h): arguments are checked here, on the host, and handed to the
// launchers as the kernels take them.  Exceptions become -1 plus the thread-local error string.
#include "../../include/shv_hip_ops.h"

#include "engine.hpp"
#include "ops.hpp"
#include "sched.hpp"

#include <cmath>
#include <cstring>
#include <stdexcept>
#include <string>

namespace {

template <class F> int guarded(F&& f) {
    try {
        f();
        return 0;
    } catch (const std::exception& e) {
        shv::sched::set_error(e.what());
        return -1;
    } catch (...) {
        shv::sched::set_error("unknown error");
        return -1;
    }
}

void require(bool ok, const char* what) {
    if (!ok) throw std::runtime_error(what);
}

shv::OpType type_of(const char* mode) {
    require(mode != nullptr, "unknown mode (fp32, bf16, fp16)");
    if (!std::strcmp(mode, "fp32")) return shv::OpType::F32;
    if (!std::strcmp(mode, "fp16")) return shv::OpType::F16;
    if (!std::strcmp(mode, "bf16")) return shv::OpType::BF16;
    throw std::runtime_error("unknown mode (fp32, bf16, fp16)");
}

size_t type_size(shv::OpType t) { return t == shv::OpType::F32 ? 4 : 2; }

void aligned_to(const void* p, size_t bytes, const char* what) {
    if (reinterpret_cast<uintptr_t>(p) % bytes) throw std::runtime_error(std::string(what) + " is not aligned to its type");
}

// A stride in elements: 0 stands for the dense one; rows may not overlap.
long long stride_or(long long s, long long dense, const char* what) {
    if (s == 0) return dense;
    if (s < dense || s > (1LL << 40)) throw std::runtime_error(std::string(what) + " out of range");
    return s;
}

// The launches of a call: an error that an earlier call of the process left behind is not this call's.
template <class F> void launch(F&& f) {
    (void)hipGetLastError();
    f();
    SHV_HIP_CHECK(hipGetLastError());
}

// ------------------------------------------------------------------------------------------ norms around a block
shv::OpType norm_args(const shv_hip_norm_args* a, shv::NormFwd* f) {
    require(a != nullptr, "null argument");
    const shv::OpType t = type_of(a->mode);
    const size_t ts = type_size(t), rs = a->residual_fp32 ? 4 : ts;
    require(a->rows >= 0 && a->rows <= (1LL << 40), "row count out of range");
    require(a->n >= 1 && a->n <= shv::kNormMaxN, "row width out of range (1..8192)");
    require(std::isfinite(a->eps) && a->eps > 0.0f, "eps has to be positive and finite");
    require(std::isfinite(a->scale), "scale has to be finite");
    if (a->gate) require(a->act >= SHV_HIP_GATE_NONE && a->act <= SHV_HIP_GATE_SIGMOID, "unknown gate activation");
    aligned_to(a->x, ts, "x");
    aligned_to(a->post_w, 4, "post_w");
    aligned_to(a->gate, a->gate_vector ? 4 : ts, "gate");
    aligned_to(a->residual, rs, "residual");
    aligned_to(a->pre_w, 4, "pre_w");
    aligned_to(a->h, rs, "h");
    aligned_to(a->y, ts, "y");
    f->rows = a->rows;
    f->n = a->n;
    f->act = a->act;
    f->gate_mode = !a->gate ? shv::GATE_ABSENT : a->gate_vector ? shv::GATE_VECTOR : shv::GATE_ROWS;
    f->res_f32 = a->residual_fp32 != 0;
    f->scale = a->scale;
    f->eps = a->eps;
    f->x = a->x;
    f->post_w = a->post_w;
    f->gate = a->gate;
    f->residual = a->residual;
    f->pre_w = a->pre_w;
    f->h = a->h;
    f->y = a->y;
    f->x_stride = stride_or(a->x_stride, a->n, "x_stride");
    f->gate_stride = stride_or(a->gate_stride, a->n, "gate_stride");
    f->residual_stride = stride_or(a->residual_stride, a->n, "residual_stride");
    f->h_stride = stride_or(a->h_stride, a->n, "h_stride");
    f->y_stride = stride_or(a->y_stride, a->n, "y_stride");
    return t;
}

size_t norm_work_bytes(const shv::NormFwd& f) {
    return size_t(3) * size_t(shv::norm_bwd_groups(f.rows, f.n)) * size_t(f.n) * sizeof(float);
}

// ------------------------------------------------------------------------------------------ the gated delta rule
constexpr const char* kTooMany = "too many sequences, heads or tokens for one call";
shv::OpType delta_args(const shv_hip_delta_args* a, shv::DeltaOp* d) {
    require(a != nullptr, "null argument");
    const shv::OpType t = type_of(a->mode);
    const size_t ts = type_size(t);
    require(a->n_seqs >= 1 && a->n_seqs <= (1 << 24), "sequence count out of range");
    require(a->heads >= 1 && a->heads <= 65535 && a->heads_qk >= 1, "head count out of range");
    require(a->heads % a->heads_qk == 0, "heads is not a multiple of heads_qk");
    require(a->dim_k >= 1 && a->dim_k <= shv::kDeltaMaxK, "dim_k out of range (1..128)");
    require(a->dim_v >= 1 && a->dim_v <= shv::kDeltaMaxV, "dim_v out of range (1..256)");
    require(a->n_tokens >= 0 && a->n_tokens <= (1LL << 36), "token count out of range");
    require(a->max_len >= 0, "max_len out of range");
    require(a->d_offsets || a->n_tokens % a->n_seqs == 0, "without offsets, n_tokens has to be a multiple of n_seqs");
    require((long long)a->n_seqs * a->heads * 16 < (1LL << 31) && a->n_tokens / 32 + a->n_seqs < (1LL << 31),
            kTooMany);
    require(std::isfinite(a->scale), "scale has to be finite");
    require(a->n_states >= 0, "state count out of range");
    aligned_to(a->d_offsets, 8, "d_offsets");
    aligned_to(a->q, ts, "q");
    aligned_to(a->k, ts, "k");
    aligned_to(a->v, ts, "v");
    aligned_to(a->o, ts, "o");
    aligned_to(a->g, 4, "g");
    aligned_to(a->beta, 4, "beta");
    aligned_to(a->state_in, 4, "state_in");
    aligned_to(a->state_out, 4, "state_out");
    aligned_to(a->state_index, 4, "state_index");
    *d = shv::DeltaOp{};
    d->n_seqs = a->n_seqs;
    d->hk = a->heads_qk;
    d->h = a->heads;
    d->dk = a->dim_k;
    d->dv = a->dim_v;
    d->n_states = a->n_states ? a->n_states : a->n_seqs;
    d->n_tokens = a->n_tokens;
    d->per_seq = a->n_tokens / a->n_seqs;
    d->max_len = a->max_len;
    d->offsets = a->d_offsets;
    d->q = a->q;
    d->k = a->k;
    d->v = a->v;
    d->g = a->g;
    d->beta = a->beta;
    d->o = a->o;
    // head strides of their own make layouts like [heads][tokens][dim] possible: a token's stride is then the dim
    d->q_head = stride_or(a->q_head, a->dim_k, "q_head");
    d->k_head = stride_or(a->k_head, a->dim_k, "k_head");
    d->v_head = stride_or(a->v_head, a->dim_v, "v_head");
    d->o_head = stride_or(a->o_head, a->dim_v, "o_head");
    const auto token = [](long long s, int heads, int dim, const char* what) {
        return s == 0 ? (long long)heads * dim : stride_or(s, dim, what);
    };
    d->q_stride = token(a->q_stride, a->heads_qk, a->dim_k, "q_stride");
    d->k_stride = token(a->k_stride, a->heads_qk, a->dim_k, "k_stride");
    d->v_stride = token(a->v_stride, a->heads, a->dim_v, "v_stride");
    d->o_stride = token(a->o_stride, a->heads, a->dim_v, "o_stride");
    d->g_stride = stride_or(a->g_stride, a->heads, "g_stride");
    d->beta_stride = stride_or(a->beta_stride, a->heads, "beta_stride");
    d->scale = a->scale;
    d->state_in = a->state_in;
    d->state_out = a->state_out;
    d->state_index = a->state_index;
    return t;
}

void delta_inputs(const shv::DeltaOp& d) {
    require(d.n_tokens == 0 || (d.q && d.k && d.v && d.g && d.beta), "null argument: q, k, v, g or beta");
}

// The scans' memory, in the order that it lies in `saved` (training) or the workspace.
size_t scan_bytes(const shv::DeltaSizes& s, bool train) {
    return s.records + s.starts + s.u + (train ? 2 : 1) * s.seg_m + 2 * s.seg_n;
}
// ... and the backward pass's: `saved` is only read there, so it has its own seg_n and seg_s.
size_t back_bytes(const shv::DeltaSizes& s) { return s.starts + s.u + 2 * s.seg_n; }
void scan_memory(const shv::DeltaSizes& s, void* p, shv::DeltaOp* d) {
    d->records = static_cast<unsigned char*>(p);
    d->starts = d->records + s.records;
    d->u = d->starts + s.starts;
    d->seg_m = d->u + s.u;
    d->seg_n = d->seg_m + s.seg_m;
    d->seg_s = d->seg_n + s.seg_n;
    d->seg_mt = d->seg_s + s.seg_n;
}

}  // namespace

extern "C" {

int shv_hip_gated_delta_sizes(const shv_hip_delta_args* a, int train, size_t* workspace, size_t* saved) {
    return guarded([&] {
        require(workspace && saved, "null argument");
        shv::DeltaOp d;
        const shv::OpType t = delta_args(a, &d);
        require(shv::delta_launches(t, d, train != 0), kTooMany);
        const shv::DeltaSizes s = shv::delta_sizes(t, d, train != 0);
        *workspace = train ? back_bytes(s) : shv::delta_by_token(d) ? 0 : scan_bytes(s, false);
        *saved = train ? scan_bytes(s, true) : 0;
    });
}

int shv_hip_gated_delta(const shv_hip_delta_args* a, void* stream) {
    return guarded([&] {
        shv::DeltaOp d;
        const shv::OpType t = delta_args(a, &d);
        delta_inputs(d);
        require(d.n_tokens == 0 || d.o, "null argument: o");
        const bool train = a->saved != nullptr;
        require(shv::delta_launches(t, d, train), kTooMany);
        if (train) {
            require(!d.state_in || d.state_in != d.state_out, "a call that trains cannot store over state_in");
            const shv::DeltaSizes s = shv::delta_sizes(t, d, true);
            require(a->saved_bytes >= scan_bytes(s, true), "saved too small");
            aligned_to(a->saved, 256, "saved");
            scan_memory(s, a->saved, &d);
        } else if (!shv::delta_by_token(d)) {
            const shv::DeltaSizes s = shv::delta_sizes(t, d, false);
            require(a->workspace && a->workspace_bytes >= scan_bytes(s, false), "workspace too small");
            aligned_to(a->workspace, 256, "workspace");
            scan_memory(s, a->workspace, &d);
        }
        launch([&] { shv::launch_delta_fwd(t, d, train, static_cast<hipStream_t>(stream)); });
    });
}

int shv_hip_gated_delta_backward(const shv_hip_delta_args* a, const shv_hip_delta_grads* g, void* stream) {
    return guarded([&] {
        shv::DeltaOp d;
        const shv::OpType t = delta_args(a, &d);
        const size_t ts = type_size(t);
        require(g != nullptr, "null argument");
        delta_inputs(d);
        require(d.n_tokens == 0 || (g->d_o && g->d_q && g->d_k && g->d_v && g->d_g && g->d_beta),
                "null argument: d_o, d_q, d_k, d_v, d_g or d_beta");
        // a sequence's first and last segments are worked on at the same time
        require(!g->d_state_in || g->d_state_in != g->d_state_out, "d_state_in cannot be d_state_out");
        require(shv::delta_launches(t, d, true), kTooMany);
        const shv::DeltaSizes s = shv::delta_sizes(t, d, true);
        require(a->saved != nullptr && a->saved_bytes >= scan_bytes(s, true), "saved too small");
        aligned_to(a->saved, 256, "saved");
        scan_memory(s, a->saved, &d);
        require(a->workspace && a->workspace_bytes >= back_bytes(s), "workspace too small");
        aligned_to(a->workspace, 256, "workspace");
        aligned_to(g->d_o, ts, "d_o");
        aligned_to(g->d_q, ts, "d_q");
        aligned_to(g->d_k, ts, "d_k");
        aligned_to(g->d_v, ts, "d_v");
        aligned_to(g->d_g, 4, "d_g");
        aligned_to(g->d_beta, 4, "d_beta");
        aligned_to(g->d_state_out, 4, "d_state_out");
        aligned_to(g->d_state_in, 4, "d_state_in");
        shv::DeltaGrad b{};
        b.d_o = g->d_o;
        b.d_state_out = g->d_state_out;
        b.d_q = g->d_q;
        b.d_k = g->d_k;
        b.d_v = g->d_v;
        b.d_g = g->d_g;
        b.d_beta = g->d_beta;
        b.d_state_in = g->d_state_in;
        b.ends = static_cast<unsigned char*>(a->workspace);
        b.dr = b.ends + s.starts;
        d.seg_n = b.dr + s.u;
        d.seg_s = d.seg_n + s.seg_n;
        launch([&] { shv::launch_delta_bwd(t, d, b, static_cast<hipStream_t>(stream)); });
    });
}

int shv_hip_norm_block(const shv_hip_norm_args* a, void* stream) {
    return guarded([&] {
        shv::NormFwd f{};
        const shv::OpType t = norm_args(a, &f);
        require(f.h || f.y, "neither h nor y is wanted");
        require(!f.y || f.pre_w, "y needs pre_w");
        if (f.rows == 0) return;
        require(f.x != nullptr, "null argument: x");
        launch([&] { shv::launch_norm_fwd(t, f, static_cast<hipStream_t>(stream)); });
    });
}

int shv_hip_norm_block_workspace(const shv_hip_norm_args* a, size_t* bytes) {
    return guarded([&] {
        require(bytes != nullptr, "null argument");
        shv::NormFwd f{};
        norm_args(a, &f);
        *bytes = norm_work_bytes(f);
    });
}

int shv_hip_norm_block_backward(const shv_hip_norm_args* a, const shv_hip_norm_grads* d, void* stream) {
    return guarded([&] {
        require(d != nullptr, "null argument");
        shv::NormBwd b{};
        const shv::OpType t = norm_args(a, &b.f);
        const size_t ts = type_size(t), rs = b.f.res_f32 ? 4 : ts;
        require(d->dh || d->dy, "neither dh nor dy is given");
        require(!d->dy || b.f.pre_w, "dy needs pre_w");
        require(!d->d_gate || b.f.gate, "a gradient of the gate is wanted without a gate");
        require(!d->d_residual || b.f.residual, "a gradient of the residual is wanted without a residual");
        require(!d->d_post_w || b.f.post_w, "a gradient of post_w is wanted without post_w");
        require(!d->d_pre_w || d->dy, "a gradient of pre_w is wanted without dy");
        const bool vec = b.f.gate_mode == shv::GATE_VECTOR;
        aligned_to(d->dh, rs, "dh");
        aligned_to(d->dy, ts, "dy");
        aligned_to(d->dx, ts, "dx");
        aligned_to(d->d_gate, vec ? 4 : ts, "d_gate");
        aligned_to(d->d_residual, rs, "d_residual");
        aligned_to(d->d_post_w, 4, "d_post_w");
        aligned_to(d->d_pre_w, 4, "d_pre_w");
        b.dh = d->dh;
        b.dy = d->dy;
        b.dx = d->dx;
        b.d_gate = vec ? nullptr : d->d_gate;
        b.d_gate_vec = vec ? static_cast<float*>(d->d_gate) : nullptr;
        b.d_residual = d->d_residual;
        b.d_post_w = d->d_post_w;
        b.d_pre_w = d->d_pre_w;
        b.part = static_cast<float*>(d->workspace);
        if (b.d_post_w || b.d_pre_w || b.d_gate_vec) {
            require(d->workspace != nullptr && d->workspace_bytes >= norm_work_bytes(b.f), "workspace too small");
            aligned_to(d->workspace, 256, "workspace");
        }
        require(b.f.rows == 0 || b.f.x != nullptr, "null argument: x");
        launch([&] { shv::launch_norm_bwd(t, b, static_cast<hipStream_t>(stream)); });
    });
}

}  // extern "C"
