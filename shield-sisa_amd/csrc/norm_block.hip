// The norms around a block with its gate and residual (shv_hip_norm_block), forward and backward.
//
//   p = x r1 w1 | x,  t = p a(z) | p,  h = res + c t | c t,  y = h r2 w2,   r = 1 / sqrt(mean(.^2) + eps)
//
// and with dH = dh + r2 (w2 dy - h r2 mean(w2 dy h r2)):
//
//   d_res = dH,  dt = c dH,  dz = dt p a'(z),  dp = dt a(z),  dx = r1 (w1 dp - x r1 mean(w1 dp x r1)),
//   dw2 = sum_rows dy h r2,  dw1 = sum_rows dp x r1,  dz of a gate vector = sum_rows dt p a'(z)
//
// Both passes are bound by memory: a row is read once into registers, its one or two means are taken there, and every
// output is written from there.  The backward pass recomputes h from x, z and the residual, which costs what reading h
// would and needs no saved statistics; it loads the next row before it works on this one.  Where a large copy reaches 5.2
// TB/s: 246,528 gated rows of 128 in bf16 forward 36 to 38 us, 5.0 to 5.3 TB/s; 8,192 rows of 2,048 in bf16 with an fp32
// residual 36 us forward (5.6 TB/s: the caches keep some of it) and 62 backward (4.9), 5.5 more for the sums of the weights'
// gradients.
//
// A row belongs to as many lanes as it has vectors of 8 values (16, 32 or 64 of them, or a workgroup of its own): few
// registers, many rows in flight.  With several vectors a lane and at most a wave a row, the gated rows of 128 took 44 us
// and a training step on the rows of 2,048 154, against 36 and 107.  The vectors need no more than their element's alignment
// (gfx950 takes any), so odd strides cost a split line, not another path: 10,272 rows of 385 in fp16 take 12 us forward (3.3
// TB/s) and 24 backward.  Narrower rows than 128 leave some of their 16 lanes without values, and the vector units, 81 % busy
// at 128, then bound: 31.6 million gated values in bf16 take 32 us in rows of 128, 49 in rows of 64, 90 of 32 and 178 of 16.
// Backward, rows of more than 4,096 take 1,024 threads of 128 registers, 10 to 12 of which spill with rows of two bytes and 57
// to 70 with fp32 ones: 15.8 million values with all parts in bf16 with an fp32 residual 95 us in rows of 4,096 (forward and
// backward), 207 in rows of 8,192.  Where 8 does not divide the row, its last lane's vector ends at the row's end and repeats
// values of the lane before: both compute and write them alike, and only the sums leave the second copy out.
#include "dev_common.hpp"
#include "ops.hpp"

#include <type_traits>

namespace shv {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float fma_of(float x, float y, float z) { return __builtin_fmaf(x, y, z); }
__device__ __forceinline__ double fma_of(double x, double y, double z) { return __builtin_fma(x, y, z); }
__device__ __forceinline__ float rsqrt_of(float x) { return __builtin_amdgcn_rsqf(x); }
__device__ __forceinline__ double rsqrt_of(double x) { return 1.0 / sqrt(x); }
__device__ __forceinline__ float rcp_of(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ double rcp_of(double x) { return 1.0 / x; }
__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

// Eight values of a row as stored: raw where a load is only issued, widened where it is used.  FEW: rows of up to 8
// values, one lane each, value by value.
template <typename T, bool FEW> struct Vec8 {
    typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    T v[8];
    __device__ __forceinline__ void load(const void* base, long long at, int c, int n, bool on) {
        const T* p = static_cast<const T*>(base) + at + c;
        if constexpr (FEW) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = on && e < n ? p[e] : T(0.0f);
        } else {
            type x = type(T(0.0f));
            if (on) x = *reinterpret_cast<const type*>(p);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = x[e];
        }
    }
    template <typename F> __device__ __forceinline__ void get(F* f) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = F(float(v[e]));
    }
    template <typename F> static __device__ __forceinline__ void store(void* base, long long at, int c, int n, bool on, const F* f) {
        T* p = static_cast<T*>(base) + at + c;
        if constexpr (FEW) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (on && e < n) p[e] = T(float(f[e]));
        } else if (on) {
            f32x8 x;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = float(f[e]);
            *reinterpret_cast<type*>(p) = __builtin_convertvector(x, type);
        }
    }
};

// a(z) and a'(z)
template <typename F> __device__ __forceinline__ F gate_act(F z, int act) {
    if (act == 0) return z;
    const F s = rcp_of(F(1) + exp_of(-z));
    return act == 1 ? z * s : s;
}
template <typename F> __device__ __forceinline__ F gate_act_d(F z, int act, F* d) {
    if (act == 0) {
        *d = 1;
        return z;
    }
    const F e = exp_of(z < 0 ? z : -z), r = rcp_of(F(1) + e), er = e * r;
    const F s = z < 0 ? er : r, ns = z < 0 ? r : er;   // sigmoid(z) and 1 - sigmoid(z), both without loss
    if (act == 1) {
        *d = s * (F(1) + z * ns);
        return z * s;
    }
    *d = s * ns;
    return s;
}

// Lanes per row: 16, 32, 64, or a workgroup of up to LPR (512, 1024)
template <int LPR> struct Lanes {
    static constexpr bool GROUP = LPR > 64;
    static constexpr int THREADS = GROUP ? LPR : kThreads, ROWS = GROUP ? 1 : kThreads / LPR, MOST = LPR * 8;
};

// Sum over the lanes of a row, the same value in each of them.  Over several waves their sums meet in LDS; two slots in
// turn, so that a wave writes a slot again only after every wave has passed the barrier behind its last read.
template <int LPR> struct RowSum {
    float (*slot)[16];   // [2][waves of the workgroup]
    int turn;
    __device__ __forceinline__ double operator()(double v) {   // (LPR = 16)
#pragma unroll
        for (int d = 1; d < 16; d *= 2) v += __shfl_xor(v, d);
        return v;
    }
    __device__ __forceinline__ float operator()(float v) {
        v = tree16(v);
        if constexpr (LPR >= 32) v = across16(v);
        if constexpr (LPR >= 64) v = across32(v);
        if constexpr (LPR > 64) {
            if ((threadIdx.x & 63) == 0) slot[turn][threadIdx.x >> 6] = v;
            __syncthreads();
            v = 0.0f;
            for (int i = 0; i < int(blockDim.x >> 6); ++i) v += slot[turn][i];
            turn ^= 1;
        }
        return v;
    }
};

// This lane's place in its row
template <int LPR, bool FEW> struct Place {
    int group, c, from;   // row of the workgroup; first column that it holds, and that is its own
    bool on, ragged;      // the lane has columns; the row's last lane repeats some
    __device__ __forceinline__ explicit Place(int n) {
        const int lane = LPR > 64 ? threadIdx.x : threadIdx.x % LPR;
        group = LPR > 64 ? 0 : threadIdx.x / LPR;
        from = 8 * lane;
        on = from < n;
        c = FEW ? 0 : from + 8 <= n ? from : n - 8;
        ragged = !FEW && (n & 7);
    }
    // a . b over the columns that are this lane's own
    template <typename F> __device__ __forceinline__ F dot(const F* a, const F* b) const {
        F s = 0;
        if (!ragged) {   // uniform over the launch
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fma_of(a[e], b[e], s);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fma_of(c + e >= from ? a[e] : F(0), b[e], s);
        }
        return s;
    }
};

// A vector's eight values of this lane over all rows: in registers, or, for 1024 threads, which have 128 of those, from
// the cache every time
template <typename F, bool FEW, bool AGAIN> struct Kept {
    const float* from;
    F v[8];
    __device__ __forceinline__ void init(const float* p, int c, int n, bool on) {
        from = p;
        if constexpr (!AGAIN) {
            Vec8<float, FEW> x;
            if (p) x.load(p, 0, c, n, on), x.get(v);
        }
    }
    __device__ __forceinline__ void get(F* x, int c, int n, bool on) const {
        if constexpr (AGAIN) {
            Vec8<float, FEW> y;
            y.load(from, 0, c, n, on);
            y.get(x);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = v[e];
        }
    }
};
// This lane's sums over its rows for a vector's gradient: in registers, or in LDS
template <bool IN_LDS> struct Sums {
    float v[8];
    __device__ __forceinline__ explicit Sums(float*) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    }
    __device__ __forceinline__ void add(const float* a, const float* b) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(a[e], b[e], v[e]);
    }
    __device__ __forceinline__ void get(float* x) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = v[e];
    }
};
template <> struct Sums<true> {
    float* p;
    __device__ __forceinline__ explicit Sums(float* lds) : p(lds + 4 * threadIdx.x) {   // 8192 floats, each lane its own
        *reinterpret_cast<f32x4*>(p) = *reinterpret_cast<f32x4*>(p + 4096) = f32x4{0, 0, 0, 0};
    }
    __device__ __forceinline__ void add(const float* a, const float* b) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 s = *reinterpret_cast<f32x4*>(p + 4096 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = __builtin_fmaf(a[4 * h + e], b[4 * h + e], s[e]);
            *reinterpret_cast<f32x4*>(p + 4096 * h) = s;
        }
    }
    __device__ __forceinline__ void get(float* x) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = p[e < 4 ? e : 4096 + e - 4];
    }
};

// T: x, gate rows and y; R: residual and h; F: what a row is computed in.
template <typename T, typename R, typename F, int LPR, bool FEW>
__global__ void __launch_bounds__(Lanes<LPR>::THREADS) norm_fwd_kernel(NormFwd a) {
    constexpr int ROWS = Lanes<LPR>::ROWS;
    __shared__ float red[2][16];
    RowSum<LPR> row_sum{red, 0};
    const Place<LPR, FEW> at(a.n);
    const F inv_n = F(1) / F(a.n);
    F w1[8], w2[8], zv[8];
    {
        Vec8<float, FEW> v;
        if (a.post_w) v.load(a.post_w, 0, at.c, a.n, at.on), v.get(w1);
        if (a.pre_w) v.load(a.pre_w, 0, at.c, a.n, at.on), v.get(w2);
        if (a.gate_mode == GATE_VECTOR) {
            v.load(a.gate, 0, at.c, a.n, at.on);
            v.get(zv);
#pragma unroll
            for (int e = 0; e < 8; ++e) zv[e] = gate_act(zv[e], a.act);
        }
    }
    for (long long first = (long long)blockIdx.x * ROWS; first < a.rows; first += (long long)gridDim.x * ROWS) {
        const long long row = first + at.group;
        const bool on = at.on && row < a.rows;   // the others compute on zeros and store nothing
        Vec8<T, FEW> x, z;
        Vec8<R, FEW> r;
        x.load(a.x, row * a.x_stride, at.c, a.n, on);
        if (a.gate_mode == GATE_ROWS) z.load(a.gate, row * a.gate_stride, at.c, a.n, on);
        if (a.residual) r.load(a.residual, row * a.residual_stride, at.c, a.n, on);
        F t[8];
        x.get(t);
        if (a.post_w) {
            const F r1 = rsqrt_of(row_sum(at.dot(t, t)) * inv_n + F(a.eps));
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = t[e] * r1 * w1[e];
        }
        if (a.gate_mode == GATE_ROWS) {
            F g[8];
            z.get(g);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] *= gate_act(g[e], a.act);
        } else if (a.gate_mode == GATE_VECTOR) {
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] *= zv[e];
        }
        if (a.residual) {
            F h[8];
            r.get(h);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = fma_of(F(a.scale), t[e], h[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] *= F(a.scale);
        }
        F s = 0;
        if (a.y) s = rsqrt_of(row_sum(at.dot(t, t)) * inv_n + F(a.eps));
        // a wave's repeated values are another's own: where h replaces the residual, every wave has read before one writes
        if (LPR > 64 && a.h == a.residual) __syncthreads();
        if (a.h) Vec8<R, FEW>::store(a.h, row * a.h_stride, at.c, a.n, on, t);
        if (a.y) {
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = t[e] * s * w2[e];
            Vec8<T, FEW>::store(a.y, row * a.y_stride, at.c, a.n, on, t);
        }
    }
}

// F is float, or double for rows of up to 8 values -- there the gradient of a norm is a difference that can cancel
// almost wholly (of one value, wholly), and what float's rounding leaves of it counts.
// A workgroup takes every gridDim-th group of rows and keeps its sums for the weights' gradients in registers; they
// are joined over its row groups in LDS and over the workgroups, in their order, by norm_sum_kernel.
template <typename T, typename R, typename F, int LPR, bool FEW>
__global__ void __launch_bounds__(Lanes<LPR>::THREADS) norm_bwd_kernel(NormBwd b) {
    constexpr int ROWS = Lanes<LPR>::ROWS, COLS = Lanes<LPR>::MOST;
    constexpr bool AHEAD = LPR < 1024;   // 1024 threads have no registers for a row in advance
    __shared__ __attribute__((aligned(16))) float keep[AHEAD ? 1 : 3 * COLS];
    __shared__ float red[2][16];
    __shared__ float fold[ROWS > 1 ? ROWS * COLS : 1];
    const NormFwd& a = b.f;
    RowSum<LPR> row_sum{red, 0};
    const Place<LPR, FEW> at(a.n);
    const int n = a.n;
    const F inv_n = F(1) / F(n);
    Kept<F, FEW, !AHEAD> w1k, w2k, zk;
    w1k.init(a.post_w, at.c, n, at.on);
    w2k.init(a.pre_w, at.c, n, at.on);
    zk.init(a.gate_mode == GATE_VECTOR ? static_cast<const float*>(a.gate) : nullptr, at.c, n, at.on);
    Sums<!AHEAD> sw1(keep), sw2(keep + (AHEAD ? 0 : COLS)), sz(keep + (AHEAD ? 0 : 2 * COLS));
    struct Row {
        Vec8<T, FEW> x, z, dy;
        Vec8<R, FEW> r, dh;
    } next;
    const auto fetch = [&](long long first) {
        const long long row = first + at.group;
        const bool on = at.on && row < a.rows;
        next.x.load(a.x, row * a.x_stride, at.c, n, on);
        if (a.gate_mode == GATE_ROWS) next.z.load(a.gate, row * a.gate_stride, at.c, n, on);
        if (b.dh) next.dh.load(b.dh, row * n, at.c, n, on);
        if (b.dy) next.dy.load(b.dy, row * n, at.c, n, on);
        if (b.dy && a.residual) next.r.load(a.residual, row * a.residual_stride, at.c, n, on);
    };
    const long long step = (long long)gridDim.x * ROWS;
    long long first = (long long)blockIdx.x * ROWS;
    if (AHEAD && first < a.rows) fetch(first);
    for (; first < a.rows; first += step) {
        if (!AHEAD) fetch(first);
        const long long row = first + at.group;
        const bool on = at.on && row < a.rows;
        const Row now = next;
        if (AHEAD && first + step < a.rows) fetch(first + step);
        F x[8], z[8], da[8], t[8], d[8], r1 = 0;
        now.x.get(x);
        if (b.dh) now.dh.get(d);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = 0;
        if (a.gate_mode == GATE_ROWS) {   // z becomes a(z)
            now.z.get(z);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = gate_act_d(z[e], a.act, &da[e]);
        } else if (a.gate_mode == GATE_VECTOR) {
            zk.get(z, at.c, n, at.on);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = gate_act_d(z[e], a.act, &da[e]);
        }
        if (a.post_w) {   // x becomes x r1
            r1 = rsqrt_of(row_sum(at.dot(x, x)) * inv_n + F(a.eps));
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= r1;
        }
        if (b.dy) {       // t is h, then h r2; d becomes dH
            F dy[8], r[8], w1[8], w2[8];
            now.dy.get(dy);
            if (a.residual) now.r.get(r);
            if (a.post_w) w1k.get(w1, at.c, n, at.on);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                F p = a.post_w ? x[e] * w1[e] : x[e];
                if (a.gate_mode != GATE_ABSENT) p *= z[e];
                t[e] = a.residual ? fma_of(F(a.scale), p, r[e]) : F(a.scale) * p;
            }
            const F r2 = rsqrt_of(row_sum(at.dot(t, t)) * inv_n + F(a.eps));
            w2k.get(w2, at.c, n, at.on);
            float p[8], q[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                t[e] *= r2;
                p[e] = float(dy[e]);
                q[e] = float(t[e]);
                dy[e] *= w2[e];
            }
            sw2.add(p, q);
            const F mean = row_sum(at.dot(dy, t)) * inv_n;
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] += r2 * (dy[e] - t[e] * mean);
        }
        // in place, every wave has read its values of this row before one is written
        if (LPR > 64 && (b.d_residual == b.dh || b.dx == b.dy)) __syncthreads();
        if (b.d_residual) Vec8<R, FEW>::store(b.d_residual, row * n, at.c, n, on, d);
        // d becomes dt, then dp (and t dz)
        F w1[8];
        if (a.post_w) w1k.get(w1, at.c, n, at.on);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] *= F(a.scale);
        if (a.gate_mode != GATE_ABSENT) {
            float p[8], q[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const F in = a.post_w ? x[e] * w1[e] : x[e];
                t[e] = d[e] * in * da[e];
                p[e] = float(d[e] * in);
                q[e] = float(da[e]);
                d[e] *= z[e];
            }
            if (a.gate_mode == GATE_VECTOR) sz.add(p, q);
        }
        if (a.post_w) {
            float p[8], q[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = float(d[e]);
                q[e] = float(x[e]);
                d[e] *= w1[e];
            }
            sw1.add(p, q);
        }
        if (b.d_gate) Vec8<T, FEW>::store(b.d_gate, row * n, at.c, n, on, t);
        if (a.post_w) {
            const F mean = row_sum(at.dot(d, x)) * inv_n;
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = r1 * (d[e] - x[e] * mean);
        }
        if (b.dx) Vec8<T, FEW>::store(b.dx, row * n, at.c, n, on, d);
    }
    const bool want[3] = {b.d_post_w != nullptr, b.d_pre_w != nullptr, b.d_gate_vec != nullptr};
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        if (!want[q]) continue;
        float v[8];
        if (q == 0) sw1.get(v);
        else if (q == 1) sw2.get(v);
        else sz.get(v);
        float* out = b.part + ((long long)q * gridDim.x + blockIdx.x) * n;
        if constexpr (ROWS > 1) {
            if (at.on)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (at.c + e < n) fold[at.group * COLS + at.c + e] = v[e];   // (a repeated column's sum is the same)
            __syncthreads();
            for (int c = threadIdx.x; c < n; c += kThreads) {
                float s = 0.0f;
#pragma unroll
                for (int g = 0; g < ROWS; ++g) s += fold[g * COLS + c];
                out[c] = s;
            }
            __syncthreads();
        } else {
            if (at.on)
#pragma unroll
                for (int e = 0; e < 8; ++e) out[at.c + e] = v[e];   // (a repeated column's sum is the same)
        }
    }
}

// [3][groups][n] -> the wanted [n]: 16 columns of one gradient per workgroup, 64 threads a column, joined in order
__global__ void __launch_bounds__(1024) norm_sum_kernel(const float* part, int groups, int n, float* d0, float* d1, float* d2) {
    __shared__ float fold[64][17];
    float* out = blockIdx.y == 0 ? d0 : blockIdx.y == 1 ? d1 : d2;
    if (!out) return;
    const int col = threadIdx.x & 15, g0 = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
    const float* p = part + (long long)blockIdx.y * groups * n;
    float s = 0.0f;
    if (c < n)
        for (int g = g0; g < groups; g += 64) s += p[(long long)g * n + c];
    fold[g0][col] = s;
    __syncthreads();
    if (threadIdx.x < 16 && c < n) {
        s = 0.0f;
        for (int g = 0; g < 64; ++g) s += fold[g][col];
        out[c] = s;
    }
}

// f(lanes per row, rows of up to 8 values)
template <class F> void for_width(int n, F&& f) {
    if (n <= 8) f(std::integral_constant<int, 16>{}, std::true_type{});
    else if (n <= 128) f(std::integral_constant<int, 16>{}, std::false_type{});
    else if (n <= 256) f(std::integral_constant<int, 32>{}, std::false_type{});
    else if (n <= 512) f(std::integral_constant<int, 64>{}, std::false_type{});
    else if (n <= 4096) f(std::integral_constant<int, 512>{}, std::false_type{});
    else f(std::integral_constant<int, 1024>{}, std::false_type{});
}
// The hardware's root takes a subnormal sum, which only a subnormal eps leaves of a row, for zero: its kernels get the least
// normal number instead.  (To scale such a sum in the kernel took the gated rows of 128 from 36.2 to 37.9 us, two runs of each in turn.)
template <typename F> float eps_for(float eps) { return std::is_same_v<F, double> || eps > 0x1p-126f ? eps : 0x1p-126f; }
// threads of a workgroup, and its rows
int threads_for(int n) { return n <= 512 ? kThreads : (n + 511) / 512 * 64; }
int rows_per_group(int n) { return n <= 128 ? 16 : n <= 256 ? 8 : n <= 512 ? 4 : 1; }
// f(T, R)
template <class F> void for_types(OpType t, bool res_f32, F&& f) {
    if (t == OpType::F32) f(float{}, float{});
    else if (t == OpType::F16 && res_f32) f(f16{}, float{});
    else if (t == OpType::F16) f(f16{}, f16{});
    else if (res_f32) f(bf16{}, float{});
    else f(bf16{}, bf16{});
}

}  // namespace

int norm_bwd_groups(long long rows, int n) {   // as many as are resident at two waves a SIMD, and at least four rows each
    const long long per = rows_per_group(n), all = (rows + per - 1) / per, waves = threads_for(n) / 64;
    const long long most = waves <= 8 ? 256 * (8 / waves) : 256;
    return int(all < 4 ? 1 : all / 4 < most ? all / 4 : most);
}

void launch_norm_fwd(OpType t, NormFwd a, hipStream_t s) {
    for_types(t, a.res_f32, [&](auto type, auto res) {
        for_width(a.n, [&](auto lpr, auto few) {
            const int threads = threads_for(a.n), rows = rows_per_group(a.n);
            typedef std::conditional_t<few.value, double, float> F;
            a.eps = eps_for<F>(a.eps);
            const long long all = (a.rows + rows - 1) / rows;
            norm_fwd_kernel<decltype(type), decltype(res), F, lpr.value, few.value>
                <<<dim3(unsigned(all < 8192 ? all : 8192)), dim3(threads), 0, s>>>(a);
        });
    });
}

void launch_norm_bwd(OpType t, NormBwd b, hipStream_t s) {
    const int groups = norm_bwd_groups(b.f.rows, b.f.n);
    for_types(t, b.f.res_f32, [&](auto type, auto res) {
        for_width(b.f.n, [&](auto lpr, auto few) {
            typedef std::conditional_t<few.value, double, float> F;
            b.f.eps = eps_for<F>(b.f.eps);
            norm_bwd_kernel<decltype(type), decltype(res), F, lpr.value, few.value>
                <<<dim3(groups), dim3(threads_for(b.f.n)), 0, s>>>(b);
        });
    });
    if (b.d_post_w || b.d_pre_w || b.d_gate_vec)
        norm_sum_kernel<<<dim3((b.f.n + 15) / 16, 3), dim3(1024), 0, s>>>(b.part, groups, b.f.n, b.d_post_w, b.d_pre_w, b.d_gate_vec);
}

}  // namespace shv
