// The operators of include/shv_hip_ops.h: arguments as the kernels take them, and their launchers.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace shv {

enum class OpType { F32, F16, BF16 };

#ifdef __HIPCC__
// v of this lane plus v of the lane 16 (32) across: one swap of odd with even rows (of halves) of two copies, and an
// addition.  In asm, since the compiler's builtin gives the first result twice; the wait states are those that it puts
// between a vector instruction and a swap.  Not for results of the matrix cores, whose wait states it would not add.
__device__ __forceinline__ float across16(float v) {
    float a = v, b = v;
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return a + b;
}
__device__ __forceinline__ float across32(float v) {
    float a = v, b = v;
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return a + b;
}
#endif

// ---- norms around a block (norm_block.hip)
enum GateMode { GATE_ABSENT = 0, GATE_ROWS = 1, GATE_VECTOR = 2 };

struct NormFwd {
    long long rows;
    int n, act, gate_mode, res_f32;
    float scale, eps;
    const void* x;
    const float* post_w;
    const void* gate;
    const void* residual;
    const float* pre_w;
    void* h;
    void* y;
    long long x_stride, gate_stride, residual_stride, h_stride, y_stride;
};

struct NormBwd {
    NormFwd f;
    const void *dh, *dy;
    void *dx, *d_gate, *d_residual;
    float *d_post_w, *d_pre_w, *d_gate_vec;
    float* part;   // [3][norm_bwd_groups][n]: per workgroup sums for post_w, pre_w and a gate vector
};

constexpr int kNormMaxN = 8192;
int norm_bwd_groups(long long rows, int n);
void launch_norm_fwd(OpType t, NormFwd a, hipStream_t s);
void launch_norm_bwd(OpType t, NormBwd a, hipStream_t s);

// ---- the gated delta rule (gated_delta.hip)
constexpr int kDeltaMaxK = 128, kDeltaMaxV = 256;

struct DeltaOp {
    int n_seqs, hk, h, dk, dv, n_states;
    long long n_tokens, per_seq, max_len;   // per_seq: tokens of each sequence where offsets is NULL
    const long long* offsets;
    const void *q, *k, *v;
    const float *g, *beta;
    void* o;
    long long q_stride, q_head, k_stride, k_head, v_stride, v_head, o_stride, o_head, g_stride, beta_stride;
    float scale;
    const float* state_in;
    float* state_out;
    const int* state_index;
    // work memory: a record per (chunk, head) from the chunks' own kernel; for training also the state that each chunk
    // starts from and every token's u, as matrix-core fragments
    unsigned char *records, *starts, *u;
    // sequences cut into segments of this many chunks: the segments' transitions M and N and the states between them
    long long segment;
    unsigned char *seg_m, *seg_mt, *seg_n, *seg_s;   // (seg_mt: M^T, for training; a backward call has seg_n, seg_s of its own)
};

struct DeltaGrad {
    const void* d_o;
    const float* d_state_out;
    void *d_q, *d_k, *d_v;
    float *d_g, *d_beta, *d_state_in;
    unsigned char *ends, *dr;   // work memory, laid out as starts and u: the gradient of the state that each chunk ends
                                // in, and T^T dU
};

struct DeltaSizes {   // bytes; starts and u are also those of the backward pass's ends and dr, seg_n that of seg_s, seg_m
                      // for training that of seg_mt
    size_t records, starts, u, seg_m, seg_n;
};
DeltaSizes delta_sizes(OpType t, const DeltaOp& a, bool train);
bool delta_by_token(const DeltaOp& a);   // the recurrent kernel serves this call: no work memory
bool delta_launches(OpType t, DeltaOp a, bool train);   // the call's launches are no larger than HIP takes
void launch_delta_fwd(OpType t, DeltaOp a, bool train, hipStream_t s);
void launch_delta_bwd(OpType t, DeltaOp a, const DeltaGrad& d, hipStream_t s);

}  // namespace shv
