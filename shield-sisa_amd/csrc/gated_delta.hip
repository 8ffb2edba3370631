// The gated delta rule (shv_hip_gated_delta): per sequence and head, with a_t = exp(g_t),
//
//   u_t = b_t (v_t - a_t S_{t-1}^T k_t),   S_t = a_t S_{t-1} + k_t u_t^T,   o_t = c S_t^T q_t
//
// In chunks of C tokens, with G_i the sum of g over the chunk's tokens up to i, S the state before the chunk, and
// D_ij = exp(G_i - G_j) for j <= i, the recurrence unrolls to
//
//   (I + L) U = diag(b) (V - diag(exp G) K S),   L_ij = b_i D_ij (k_i . k_j) for j < i
//   O = c diag(exp G) Q S + A U,                 A_ij = c D_ij (q_i . k_j) for j <= i
//   S' = exp(G_C) S + K^T diag(exp(G_C - G)) U
//
// T = (I + L)^-1 and A depend on no state: delta_chunk_kernel computes them for all chunks at once and leaves them as
// matrix-core fragments (a "record" per chunk and head).  delta_scan_kernel then walks a sequence's chunks; the columns
// of S, V, U and O do not mix, so a wave owns 16 of them and carries its part of S in registers.
//
// Every product runs on v_mfma_f32_16x16x32_bf16 with operands split into bf16 parts, fp32 sums: inputs exactly (bf16
// one part, fp16 two, fp32 three), what is computed on the way -- S, U, T, A -- as three parts, fp32's own precision.
// That holds for what reaches only an fp16 or bf16 o as well: where a token replaces what its key held, Q S and A U
// cancel, and what two parts leave out (2^-17 of them) is then no longer below o's own rounding.  bf16 parts have fp32's
// range, so nothing is scaled.
//
// Fragment orders.  The contraction index of a product may be visited in any order as long as both operands agree.  A
// result fragment holds, per lane (g, r), column r and rows 4 g .. 4 g + 3 of a 16-row tile; an operand fragment wants
// eight consecutive contraction indices 8 g .. 8 g + 7 of 32.  Two 16-row tiles i = 2 p, 2 p + 1 therefore stand for the
// rows 32 p + 8 g + 4 (i & 1) + e (e = 0..3): what one product leaves in registers is then the next one's operand as it
// is -- S, R, U and their gradients never pass through LDS.
#include "dev_common.hpp"
#include "ops.hpp"

#include <type_traits>

namespace shv {
namespace {

typedef float f32x8v __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Parts;            // bf16 parts of an input; tokens per chunk
template <> struct Parts<bf16> { static constexpr int IN = 1, C = 64; };
template <> struct Parts<f16> { static constexpr int IN = 2, C = 64; };
template <> struct Parts<float> { static constexpr int IN = 3, C = 32; };
constexpr int MID = 3;                         // bf16 parts of everything else

constexpr int kBlock = 1024;   // bytes of a 16 x 32 fragment block

// 16-byte slot of (row r, contraction octet c) in a fragment block: lane-contiguous rows for the loads that fill it,
// and the 16 lanes of an operand read on 16 distinct bank groups
__device__ __forceinline__ int slot_of(int r, int c) { return 4 * r + (c ^ (((r >> 2) ^ (r >> 1)) & 3)); }
// row r of 16-row tile i, as an index of the 32-row pair that it belongs to
__device__ __forceinline__ int row_of(int i, int r) { return 32 * (i >> 1) + 8 * (r >> 2) + 4 * (i & 1) + (r & 3); }
// block (i, s) of a lower triangular matrix: row tiles of pair p = i >> 1 hold the contraction blocks s <= p
__device__ __forceinline__ constexpr int tri(int i, int s) { return (i >> 1) * ((i >> 1) + 1) + (i & 1) * ((i >> 1) + 1) + s; }
// ... and of an upper triangular one: row tile i holds the contraction blocks s >= i >> 1
__device__ __forceinline__ constexpr int tri_up(int i, int s) { return s * (s + 1) + i; }

template <typename T> struct Record {   // what delta_chunk_kernel leaves per (chunk, head): T^T, vectors, A^T
    static constexpr int C = Parts<T>::C, NT = C / 16, NP = C / 32, BLOCKS = NP * (NP + 1), MAT = BLOCKS * kBlock;
    static constexpr int VEC_AT = MID * MAT, A_AT = VEC_AT + kBlock;   // vectors: exp G, exp(G_C - G), b, C floats each; exp G_C
    static constexpr int BYTES = A_AT + MID * MAT;
    static_assert(3 * C * 4 + 16 <= kBlock, "the vectors' block");
};

// x = the sum of its parts, each the rounding of what the earlier ones leave; two values at a time, so that a pair's
// part is one packed conversion and is widened again from where it lies
template <int P> __device__ __forceinline__ void split8(const float* x, bf16x8* part) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    u32x4 out[P];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f32x2 rest = {x[2 * e], x[2 * e + 1]};
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const unsigned h = __builtin_bit_cast(unsigned, __builtin_convertvector(rest, bf16x2));
            out[p][e] = h;
            if (p + 1 < P) rest = f32x2{rest[0] - __builtin_bit_cast(float, h << 16), rest[1] - __builtin_bit_cast(float, h & 0xffff0000u)};
        }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) part[p] = __builtin_bit_cast(bf16x8, out[p]);
}
template <int P> __device__ __forceinline__ void split8(f32x4 lo, f32x4 hi, bf16x8* part) {
    const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    split8<P>(x, part);
}

// The pairs of parts whose product reaches 2^-8P of the leading one, smallest first: f(part of a, part of b).
template <int PA, int PB, class F> __device__ __forceinline__ void for_pairs(F&& f) {
    constexpr int P = PA > PB ? PA : PB;
#pragma unroll
    for (int sum = P - 1; sum >= 0; --sum)
#pragma unroll
        for (int i = PA - 1; i >= 0; --i)
            if (sum - i >= 0 && sum - i < PB) f(i, sum - i);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
// c[n] += a[n] b, and with the operands' places exchanged c[n] += b a[n]; N sums side by side, so that an MFMA does not
// wait for the one before it
template <int N, int PA, int PB> __device__ __forceinline__ void mul(const bf16x8 (&a)[N][PA], const bf16x8 (&b)[PB], f32x4* c) {
    for_pairs<PA, PB>([&](int i, int j) {
#pragma unroll
        for (int n = 0; n < N; ++n) c[n] = mfma(a[n][i], b[j], c[n]);
    });
}
template <int N, int PA, int PB> __device__ __forceinline__ void mul_t(const bf16x8 (&b)[PB], const bf16x8 (&a)[N][PA], f32x4* c) {
    for_pairs<PA, PB>([&](int i, int j) {
#pragma unroll
        for (int n = 0; n < N; ++n) c[n] = mfma(b[j], a[n][i], c[n]);
    });
}
// Loads stay above this and what uses them below: the compiler otherwise sinks each LDS read to its use and waits there.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }
// Between two fences: N times one MFMA and then V vector instructions, so that the vector unit works while the matrix
// core does (an MFMA takes it 16 cycles, a vector instruction 4); READS LDS reads go first.
template <int N, int V, int READS = 0> __device__ __forceinline__ void interleave() {
    if constexpr (READS > 0) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
    }
}

template <typename T> struct Loose8 { typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T)))); };
template <typename T> struct Loose4 { typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T)))); };

// values at .. at + 7 of a row of n (zeros past its end), as stored
template <typename T> __device__ __forceinline__ typename Loose8<T>::type load8(const T* row, int at, int n) {
    if (at + 8 <= n) return *reinterpret_cast<const typename Loose8<T>::type*>(row + at);
    typename Loose8<T>::type v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = at + e < n ? row[at + e] : T(0.0f);
    return v;
}

// A sequence's tokens; offsets are clamped so that nothing that they hold leads outside the buffers.
__device__ __forceinline__ long long seq_begin(const DeltaOp& a, int i) {
    if (!a.offsets) return a.per_seq * i;
    const long long b = a.offsets[i];
    return b < 0 ? 0 : b > a.n_tokens ? a.n_tokens : b;
}
__device__ __forceinline__ long long seq_len(const DeltaOp& a, int i, long long begin) {
    if (!a.offsets) return a.per_seq;
    const long long n = seq_begin(a, i + 1) - begin;
    return n < 0 ? 0 : n;
}
__device__ __forceinline__ int state_of(const DeltaOp& a, int seq) {
    const int i = a.state_index ? a.state_index[seq] : seq;
    return i >= 0 && i < a.n_states ? i : -1;
}
// g's sum stays finite, so that differences across a reset (g = -inf) are -1e5 or less and their exp is 0; NaN stays
// ... in units of log 2, so that exp is one hardware exp2 of a difference that double has taken exactly
__device__ __forceinline__ double log_decay(float g) { return 1.4426950408889634074 * (g < -1e5f ? -1e5 : double(g)); }
__device__ __forceinline__ float decay_of(double g) { return __builtin_amdgcn_exp2f(float(g)); }

// Piece c (of `size` tokens: chunks, segments) of a sequence that begins at token b has slot b / size + seq + c: slots
// are distinct, since a sequence of n tokens ends below slot (b + n) / size + seq + 1.  An empty sequence has piece 0.
struct Piece {
    int seq;
    long long begin, len, c;   // the sequence's first token and length; the piece's number
};
__device__ __forceinline__ long long quotient(long long x, long long y) {   // x >= 0, y > 0
    return (x | y) >> 32 ? x / y : (long long)(unsigned(x) / unsigned(y));
}
// By all lanes of a wave: 64 sequences are looked at at a time, one load deep where a binary search would wait for six.
__device__ __forceinline__ bool piece_of(const DeltaOp& a, long long slot, long long size, Piece* p) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = a.n_seqs - 1;
    while (lo < hi) {   // the last sequence whose first slot is not past this one
        const int step = (hi - lo) / 64 + 1, i = hi - lo < lane * (long long)step ? hi : lo + lane * step;
        const bool before = lo + lane * (long long)step <= hi && quotient(seq_begin(a, i), size) + i <= slot;
        const int found = __builtin_popcountll(__ballot(before));
        lo += (found > 0 ? found - 1 : 0) * step;
        hi = lo + step - 1 < hi ? lo + step - 1 : hi;
    }
    p->seq = lo;
    p->begin = seq_begin(a, lo);
    p->len = seq_len(a, lo, p->begin);
    p->c = slot - quotient(p->begin, size) - lo;
    return p->c == 0 || (p->c > 0 && p->c * size < p->len);
}
// Workgroups go round-robin over the eight XCDs, each with an L2 of its own.  So an XCD gets a contiguous eighth of the
// work in the order (q / k head, slot, value head of its group, slice): what shares rows of q and k, a record or a
// transition, and what one kernel leaves for the next, then meets in one L2.
struct Item {
    long long slot;
    int head, slice;
};
constexpr int kXcds = 8;
__device__ __forceinline__ bool item_of(const DeltaOp& a, long long slots, int heads, int slices, Item* it) {
    const int group = heads / a.hk;
    const unsigned n = unsigned(slots * heads * slices), per = (n + kXcds - 1) / kXcds;   // (delta_launches keeps it small)
    unsigned id = blockIdx.x % kXcds * per + blockIdx.x / kXcds;
    if (blockIdx.x / kXcds >= per || id >= n) return false;
    it->slice = int(id % unsigned(slices));
    id /= unsigned(slices);
    const int member = int(id % unsigned(group));
    id /= unsigned(group);
    it->slot = id % unsigned(slots);
    it->head = int(id / unsigned(slots)) * group + member;
    return true;
}
__device__ __forceinline__ long long slots_of(const DeltaOp& a, long long tokens) { return a.n_tokens / tokens + a.n_seqs; }

template <int C> __device__ __forceinline__ bool chunk_of(const DeltaOp& a, long long slot, int* seq, long long* begin, int* valid) {
    Piece p;
    if (!piece_of(a, slot, C, &p) || p.c * C >= p.len) return false;
    *seq = p.seq;
    *begin = p.begin + p.c * C;
    *valid = p.len - p.c * C < C ? int(p.len - p.c * C) : C;
    return true;
}

// The C rows of one head of q or k, 16 bytes of T at a time: UNITS loads per thread, then as many slots of the
// fragment tile [part][row tile][contraction block].  WHOLE: every row has all 32 NK values and is aligned, offsets fit
// 32 bits; rows past the last token then repeat it (their b is 0, so they take part in nothing), else they are zeros.
template <typename T, int NK, int THREADS> struct RowTile {
    static constexpr int C = Parts<T>::C, NT = C / 16, P = Parts<T>::IN, BYTES = P * NT * NK * kBlock;
    static constexpr int UNITS = (NT * NK * 64 + THREADS - 1) / THREADS;
    typename Loose8<T>::type raw[UNITS];
    static __device__ __forceinline__ int row_in(int u) { return row_of((u >> 6) / NK, (u & 63) >> 2); }
    static __device__ __forceinline__ int col_in(int u) {
        const int r = (u & 63) >> 2;
        return 32 * ((u >> 6) % NK) + 8 * ((u & 3) ^ (((r >> 2) ^ (r >> 1)) & 3));
    }
    template <bool WHOLE>
    __device__ __forceinline__ void load(const T* base, long long stride, int valid, int d, int tid) {
#pragma unroll
        for (int n = 0; n < UNITS; ++n) {
            const int u = tid + n * THREADS, t = row_in(u), x = col_in(u);
            if constexpr (WHOLE) {
                const unsigned off = unsigned(t < valid ? t : valid - 1) * unsigned(stride) + unsigned(x);
                if (NT * NK * 64 % THREADS == 0 || u < NT * NK * 64)
                    raw[n] = *reinterpret_cast<const typename Row8<T>::type*>(base + off);
            } else {
                const bool in = u < NT * NK * 64 && t < valid && x < d;
                raw[n] = load8(base + (in ? t * stride : 0), in ? x : 0, in ? d : 0);
            }
        }
    }
    __device__ __forceinline__ void store_raw(unsigned char* tile, int tid) const {   // two-byte types as they are
#pragma unroll
        for (int n = 0; n < UNITS; ++n) {
            const int u = tid + n * THREADS;
            if (NT * NK * 64 % THREADS && u >= NT * NK * 64) break;
            *reinterpret_cast<typename Row8<T>::type*>(tile + (u >> 6) * kBlock + (u & 63) * 16) = raw[n];
        }
    }
    __device__ __forceinline__ void store(unsigned char* tile, int tid) const {
#pragma unroll
        for (int n = 0; n < UNITS; ++n) {
            const int u = tid + n * THREADS;
            if (NT * NK * 64 % THREADS && u >= NT * NK * 64) break;
            bf16x8 part[P];
            if constexpr (P == 1) {
                part[0] = __builtin_bit_cast(bf16x8, raw[n]);
            } else {
                const f32x8 x = __builtin_convertvector(raw[n], f32x8);
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = x[e];
                split8<P>(y, part);
            }
#pragma unroll
            for (int p = 0; p < P; ++p)
                *reinterpret_cast<bf16x8*>(tile + p * (NT * NK * kBlock) + (u >> 6) * kBlock + (u & 63) * 16) = part[p];
        }
    }
};

// LDS by its own addresses: one base per tile and lane, everything else an immediate offset
typedef __attribute__((address_space(3))) unsigned char* Lds;
typedef __attribute__((address_space(3))) bf16x8* LdsFrag;
typedef __attribute__((address_space(3))) s16x4* LdsQuad;
typedef __attribute__((address_space(3))) f32x4* LdsVec;

// Operand fragment of block `blk` of a tile with P parts `stride` bytes apart; the base includes the lane's
// 16 slot_of(r, g).
template <int P> __device__ __forceinline__ void read_frag(Lds tile, int stride, int blk, bf16x8 (&f)[P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) f[p] = *(LdsFrag)(tile + p * stride + blk * kBlock);
}
// Operand fragment of the tile's transpose: row tile m of its columns, contraction block s over its rows.  The 16 lanes
// of a group hand the transposing read four rows x 16 columns, each lane one row's four; the base includes the lane's
// 16 slot_of(4 g + (r >> 2), r & 3).  `blk(i)` is the block of row tile i and column block m >> 1.
template <int P, class F>
__device__ __forceinline__ void read_frag_t(Lds tile, int stride, F&& blk, int m, int s, bf16x8 (&f)[P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
        union { s16x4 q[2]; bf16x8 v; } x;
#pragma unroll
        for (int half = 0; half < 2; ++half)
            x.q[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsQuad)(tile + p * stride + blk(2 * s + half) * kBlock + 8 * (m & 1)));
        f[p] = x.v;
    }
}
// a fragment to global memory, as a block per part
template <int P> __device__ __forceinline__ void store_frag(unsigned char* to, int at, const bf16x8 (&f)[P]) {
#pragma unroll
    for (int p = 0; p < P; ++p) *reinterpret_cast<bf16x8*>(to + p * kBlock + at) = f[p];
}

// ------------------------------------------------------------------------------------------ chunks on their own
__device__ __forceinline__ void copy_lds16(const void* src, void* lds_block) {
    __builtin_amdgcn_global_load_lds(src, lds_block, 16, 0, 0);
}
__device__ __forceinline__ void arrive() {   // what this wave fetched and stored to LDS is there, for every wave
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Rows of q and k against rows of k, on the matrix cores of their own type: products of inputs are exact there, so the
// two-byte types need one tile each, as stored.
template <typename T> struct Plain {
    static constexpr int P = 1;
    typedef T V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 mul(const V8* a, const V8* b, f32x4 c) {
        if constexpr (std::is_same_v<T, f16>) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], b[0], c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[0], c, 0, 0, 0);
    }
};
template <> struct Plain<float> {
    static constexpr int P = 3;
    typedef bf16x8 V8;
    static __device__ __forceinline__ f32x4 mul(const V8* a, const V8* b, f32x4 c) {
        for_pairs<3, 3>([&](int i, int j) { c = mfma(a[i], b[j], c); });
        return c;
    }
};

// T = (I + L)^-1 and A of one chunk and head, by four waves.  Wave j takes the columns of token tile j of K K^T and
// Q K^T: a lane then holds, for its column, eight consecutive rows of two row tiles, which are a slot of A^T's fragments
// as they are.  L goes to LDS by columns.  Its 16 x 16 diagonal blocks are inverted by forward substitution, a lane per
// column; the blocks below them column by column, T_ij = -T_ii sum_k L_ik T_kj, in fp32 on the matrix cores.
// Memory and the chain of substitutions share the time: 257 chunks x 8 heads of 128 keys in bf16 take 31 us, 38 MB read and
// 77 MB of records written, 3.7 TB/s; many small workgroups hide the chains of each other.
template <typename T, int NK, bool WHOLE>
__global__ void __launch_bounds__(256) delta_chunk_kernel(DeltaOp a) {
    typedef Record<T> R;
    typedef Plain<T> X;
    constexpr int C = R::C, NT = R::NT, NP = R::NP, P = X::P, PITCH = C + 4;
    constexpr int TILE = P * NT * NK * kBlock, COLS = C * PITCH * 4, BYTES = 2 * TILE > COLS ? 2 * TILE : COLS;
    __shared__ __attribute__((aligned(1024))) unsigned char mem[BYTES];
    __shared__ __attribute__((aligned(16))) float diag[NT][16][20];   // T's diagonal blocks, by columns
    __shared__ double gsum[C];
    __shared__ float bet[C];
    int seq, valid;
    long long begin;
    Item it;
    if (!item_of(a, slots_of(a, C), a.h, 1, &it) || !chunk_of<C>(a, it.slot, &seq, &begin, &valid)) return;   // uniform
    const int head = it.head, hq = head / (a.h / a.hk);
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    unsigned char *kt = mem, *qt = mem + TILE;
    typedef RowTile<T, NK, 256> Rows;
    const T* kp = static_cast<const T*>(a.k) + begin * a.k_stride + hq * a.k_head;
    const T* qp = static_cast<const T*>(a.q) + begin * a.q_stride + hq * a.q_head;
    if constexpr (WHOLE && P == 1) {
#pragma unroll
        for (int n = 0; n < NT * NK / 4; ++n) {
            const int u = (wave + n * 4) * 64 + lane, t = Rows::row_in(u), row = t < valid ? t : valid - 1;
            copy_lds16(kp + (unsigned(row) * unsigned(a.k_stride) + unsigned(Rows::col_in(u))), kt + (wave + n * 4) * kBlock);
            copy_lds16(qp + (unsigned(row) * unsigned(a.q_stride) + unsigned(Rows::col_in(u))), qt + (wave + n * 4) * kBlock);
        }
    }
    if (wave == 0) {   // running sum of g, a token per lane
        double s = lane < valid ? log_decay(a.g[(begin + lane) * a.g_stride + head]) : 0.0;
#pragma unroll
        for (int d = 1; d < C; d *= 2) {
            const double up = __shfl_up(s, d);
            if (lane >= d) s += up;
        }
        if (lane < C) {
            gsum[lane] = s;
            bet[lane] = lane < valid ? a.beta[(begin + lane) * a.beta_stride + head] : 0.0f;
        }
    }
    if constexpr (!(WHOLE && P == 1)) {
        Rows k, q;
        k.template load<WHOLE>(kp, a.k_stride, valid, a.dk, tid);
        q.template load<WHOLE>(qp, a.q_stride, valid, a.dk, tid);
        if constexpr (P == 1) {
            k.store_raw(kt, tid);
            q.store_raw(qt, tid);
        } else {
            k.store(kt, tid);
            q.store(qt, tid);
        }
    }
    arrive();
    // with two token tiles (C = 32) two waves take a column each and one product
    constexpr int BOTH = NT == 4 ? 2 : 1;
    const int j = wave & (NT - 1), first = NT == 4 ? 0 : wave >> 1, at = 16 * slot_of(r, g);
    f32x4 acc[BOTH][NT];
#pragma unroll
    for (int w = 0; w < BOTH; ++w)
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[w][i] = f32x4{0, 0, 0, 0};
    const auto frag = [&](const unsigned char* tile, int blk, typename X::V8* f) {
#pragma unroll
        for (int p = 0; p < P; ++p) f[p] = *reinterpret_cast<const typename X::V8*>(tile + p * (NT * NK * kBlock) + blk * kBlock + at);
    };
#pragma unroll
    for (int s = 0; s < NK; ++s) {
        typename X::V8 y[P];
        frag(kt, j * NK + s, y);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if ((i >> 1) < (j >> 1)) continue;
#pragma unroll
            for (int w = 0; w < BOTH; ++w) {
                typename X::V8 x[P];
                frag(first + w ? qt : kt, i * NK + s, x);
                acc[w][i] = X::mul(x, y, acc[w][i]);
            }
        }
    }
    __syncthreads();   // the tiles are read; their memory now holds L's columns
    float(*lt)[PITCH] = reinterpret_cast<float(*)[PITCH]>(mem);
    unsigned char* rec = a.records + (it.slot * a.h + head) * R::BYTES;
    const int col = row_of(j, r);
    const double gc = gsum[col];
#pragma unroll
    for (int s = 0; s < NP; ++s) {
        if (s < (j >> 1)) continue;
        f32x4 l[2], q[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int i = 2 * s + n, row = row_of(i, 4 * g);
            const f32x4 b = *reinterpret_cast<const f32x4*>(&bet[row]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float d = col <= row + e ? decay_of(gsum[row + e] - gc) : 0.0f;
                const float x = acc[0][i][e], y = acc[BOTH - 1][i][e];
                l[n][e] = col < row + e ? b[e] * (d * x) : 0.0f;
                q[n][e] = col <= row + e && row + e < valid ? a.scale * (d * y) : 0.0f;
            }
            if (first == 0) *reinterpret_cast<f32x4*>(&lt[col][row]) = l[n];
        }
        if (first + BOTH == 2) {
            bf16x8 part[MID];
            split8<MID>(q[0], q[1], part);
#pragma unroll
            for (int p = 0; p < MID; ++p)
                *reinterpret_cast<bf16x8*>(rec + R::A_AT + p * R::MAT + tri_up(j, s) * kBlock + at) = part[p];
        }
    }
    if (tid < C) {
        float* vec = reinterpret_cast<float*>(rec + R::VEC_AT);
        const float all = decay_of(gsum[tid]);
        vec[tid] = tid < valid ? all : 0.0f;   // a row past the last token, which repeats that token, reads nothing
        if (tid == C - 1) vec[3 * C] = all;
        vec[C + tid] = decay_of(gsum[C - 1] - gsum[tid]);
        vec[2 * C + tid] = bet[tid];
    }
    __syncthreads();
    if (NT < 4 && wave >= NT) return;   // uniform over a wave; NT waves meet at the one barrier that is left
    // T's diagonal block: lane r's column of it, the four lane groups alike
    float t[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) t[x] = x == r ? 1.0f : 0.0f;
#pragma unroll
    for (int y = 0; y < 15; ++y) {
        float l[16];
#pragma unroll
        for (int x = (y + 1) & ~3; x < 16; x += 4) *reinterpret_cast<f32x4*>(l + x) = *reinterpret_cast<const f32x4*>(&lt[16 * wave + y][16 * wave + x]);
#pragma unroll
        for (int x = y + 1; x < 16; ++x) t[x] = __builtin_fmaf(-l[x], t[y], t[x]);
    }
    f32x4 colb[NT];
#pragma unroll
    for (int e = 0; e < 4; ++e) colb[0][e] = g == 0 ? t[e] : g == 1 ? t[4 + e] : g == 2 ? t[8 + e] : t[12 + e];
    *reinterpret_cast<f32x4*>(&diag[wave][r][4 * g]) = colb[0];
    __syncthreads();
    const f32x4 own = colb[0];
    // the blocks below it
#pragma unroll
    for (int x = 0; x < NT; ++x) {
        if (x < wave) {
            colb[x] = f32x4{0, 0, 0, 0};
            continue;
        }
        if (x == wave) {
            colb[x] = own;
            continue;
        }
        f32x4 s = {0, 0, 0, 0}, z = {0, 0, 0, 0};
#pragma unroll
        for (int y = 0; y < x; ++y) {
            if (y < wave) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                s = __builtin_amdgcn_mfma_f32_16x16x4f32(lt[16 * y + 4 * g + e][16 * x + r], colb[y][e], s, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) z = __builtin_amdgcn_mfma_f32_16x16x4f32(diag[x][4 * g + e][r], s[e], z, 0, 0, 0);
        colb[x] = -z;
    }
    // T^T: row 16 wave + r of it, four contraction indices 16 x + 4 g .. of each block
    const int row = 16 * wave + r, tile = 2 * (row >> 5) + ((row >> 2) & 1), in_tile = 4 * ((row >> 3) & 3) + (row & 3);
#pragma unroll
    for (int x = 0; x < NT; ++x) {
        if ((x >> 1) < (wave >> 1)) continue;
        const int to = tri_up(tile, x >> 1) * kBlock + 16 * slot_of(in_tile, 2 * (x & 1) + (g >> 1)) + 8 * (g & 1);
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        f32x4 rest = colb[x];
#pragma unroll
        for (int p = 0; p < MID; ++p) {
            const bf16x4 h = __builtin_convertvector(rest, bf16x4);
            *reinterpret_cast<bf16x4*>(rec + p * R::MAT + to) = h;
            rest -= __builtin_convertvector(h, f32x4);
        }
    }
}

// ------------------------------------------------------------------------------------------ the scan over chunks
// What a chunk step reads, fetched a step ahead into the other of two LDS stages: the K tile, the Q tile, the columns X
// of v or d_o, the record.  Where the inputs are already what the tiles hold (bf16, WHOLE) everything goes straight to
// LDS; else K and Q wait in registers and are converted and stored when the step ends -- into the other stage, or, where
// two do not fit, into their own place behind one more barrier.  X of two bytes goes through LDS as well (the
// transposing read hands a lane four tokens of its column), X of four bytes and unaligned X through registers.  Where two
// stages of X do not fit either, it has one, and a barrier between the step's own read of it and the fetch (xs_read).
template <typename T, int NK, int W, bool WHOLE, bool WITH_Q, int REC> struct Feed {
    typedef Record<T> R;
    typedef RowTile<T, NK, 64 * W> Tile;
    static constexpr int C = R::C, NT = R::NT;
    static constexpr bool DIRECT = WHOLE && sizeof(T) == 2 && Parts<T>::IN == 1, X_LDS = WHOLE && sizeof(T) == 2;
    static constexpr int KQ = (WITH_Q ? 2 : 1) * Tile::BYTES, X_BYTES = X_LDS ? NT * (W / 2) * kBlock : 0;
    static constexpr bool TWO = DIRECT || 2 * (KQ + X_BYTES + REC) <= 160 * 1024;
    static constexpr int TILES = (TWO ? 2 : 1) * KQ;
    static constexpr bool TWO_X = TILES + 2 * (X_BYTES + REC) <= 160 * 1024;
    static constexpr int BYTES = TILES + 2 * REC + (TWO_X ? 2 : 1) * X_BYTES;
    static_assert(BYTES <= 160 * 1024, "LDS");
    unsigned char* mem;
    const T *k, *q, *x;         // the head's rows at the sequence's first token
    const unsigned char* rec;   // the head's record of the sequence's first chunk
    long long k_stride, q_stride, x_stride, rec_stride;
    long long len;
    int dk, dv, tid, col, xcol;   // xcol: first column of the workgroup's part of X
    Tile kr, qr;
    T xr[NT][4], xn[NT][4];

    __device__ __forceinline__ unsigned char* k_tile(int st) const { return mem + (TWO ? st * KQ : 0); }
    __device__ __forceinline__ unsigned char* q_tile(int st) const { return k_tile(st) + Tile::BYTES; }
    __device__ __forceinline__ unsigned char* record(int st) const { return mem + TILES + st * REC; }
    __device__ __forceinline__ unsigned char* x_tile(int st) const { return mem + TILES + 2 * REC + (TWO_X ? st * X_BYTES : 0); }

    __device__ __forceinline__ void rows(const T* base, long long stride, int valid, unsigned char* tile) const {
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
#pragma unroll
        for (int n = 0; n < (NT * NK + W - 1) / W; ++n) {
            const int u = (wave + n * W) * 64 + lane, t = Tile::row_in(u);
            if (NT * NK % W && wave + n * W >= NT * NK) break;
            copy_lds16(base + (unsigned(t < valid ? t : valid - 1) * unsigned(stride) + unsigned(Tile::col_in(u))), tile + (wave + n * W) * kBlock);
        }
    }
    // One of four pieces of chunk c's loads (K; Q; X; the record), so that a step can issue them between its products:
    // all at once they would queue in front of the address unit with every wave waiting.
    __device__ __forceinline__ void fetch_piece(int piece, long long c, int st, bool with_x) {
        const int valid = len - c * C < C ? int(len - c * C) : C;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
        const long long t0 = c * C;
        if (piece == 0) {
            if constexpr (DIRECT) rows(k + t0 * k_stride, k_stride, valid, k_tile(st));
            else kr.template load<WHOLE>(k + t0 * k_stride, k_stride, valid, dk, tid);
        } else if (piece == 1) {
            if constexpr (WITH_Q) {
                if constexpr (DIRECT) rows(q + t0 * q_stride, q_stride, valid, q_tile(st));
                else qr.template load<WHOLE>(q + t0 * q_stride, q_stride, valid, dk, tid);
            }
        } else if (piece == 2) {
            if (!with_x) return;
            const T* xp = x + t0 * x_stride;
            if constexpr (X_LDS) {
#pragma unroll
                for (int n = 0; n < NT / 2; ++n) {   // block (token tile, 32 columns); columns past dv repeat the last ones
                    const int b = wave + n * W, r = lane >> 2, t = row_of(b / (W / 2), r), c0 = xcol + 32 * (b % (W / 2));
                    const int c1 = (c0 < dv ? c0 : dv - 32) + 8 * ((lane & 3) ^ (((r >> 2) ^ (r >> 1)) & 3));
                    copy_lds16(xp + (unsigned(t < valid ? t : valid - 1) * unsigned(x_stride) + unsigned(c1)), x_tile(st) + b * kBlock);
                }
            } else {
                const int g = lane >> 4;
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = row_of(i, 4 * g + e);
                        if constexpr (WHOLE)
                            xn[i][e] = xp[unsigned(t < valid ? t : valid - 1) * unsigned(x_stride) + unsigned(col < dv ? col : 0)];
                        else
                            xn[i][e] = t < valid && col < dv ? xp[t * x_stride + col] : T(0.0f);
                    }
            }
        } else {
            const unsigned char* rp = rec + c * rec_stride + lane * 16;
#pragma unroll
            for (int n = 0; n < (REC / kBlock + W - 1) / W; ++n) {
                const int blk = wave + n * W;
                if (REC / kBlock % W == 0 || blk < REC / kBlock) copy_lds16(rp + blk * kBlock, record(st) + blk * kBlock);
            }
        }
        fence();
    }
    __device__ __forceinline__ void fetch(long long c, int st, bool with_x) {
#pragma unroll
        for (int piece = 0; piece < 4; ++piece) fetch_piece(piece, c, st, with_x);
    }
    // the X columns of the step that fetch prepared: from LDS as stored, and widened
    __device__ __forceinline__ void read_x(int st, s16x4* raw) const {
        const int lane = tid & 63, r = lane & 15, g = lane >> 4, wave = tid >> 6;
        if constexpr (X_LDS) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
                raw[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (LdsQuad)((Lds)x_tile(st) + (i * (W / 2) + (wave >> 1)) * kBlock + 16 * slot_of(4 * g + (r >> 2), r & 3) + 8 * (wave & 1)));
        }
    }
    __device__ __forceinline__ void columns(int st, f32x4* v) const {
        s16x4 raw[NT];
        read_x(st, raw);
        widen(raw, v);
    }
    __device__ __forceinline__ void widen(const s16x4* raw, f32x4* v) const {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if constexpr (X_LDS) {
                typedef T T4 __attribute__((ext_vector_type(4)));
                v[i] = __builtin_convertvector(__builtin_bit_cast(T4, raw[i]), f32x4);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[i][e] = float(xr[i][e]);
            }
        }
    }
    // Every wave has its columns of X and the next step's may take their place.  LDS alone: the loads ahead stay in flight.
    __device__ __forceinline__ void xs_read() const {
        if constexpr (!TWO_X) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    // X in registers moves on: what was fetched becomes the current step's, so that the next fetch can be issued
    __device__ __forceinline__ void advance() {
        if constexpr (!X_LDS) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) xr[i][e] = xn[i][e];
        }
    }
    // the end of a step: the next one's tiles are in LDS
    __device__ __forceinline__ void commit(int st, bool more) {
        if constexpr (!DIRECT) {
            if (!TWO) __syncthreads();   // every wave is done with the tiles
            if (more) {
                kr.store(k_tile(st), tid);
                if constexpr (WITH_Q) qr.store(q_tile(st), tid);
            }
        }
        arrive();
    }
};

// A state's columns of one wave, as its accumulators hold them: 16 bytes per lane and tile
template <int M> __device__ __forceinline__ void load_acc(const unsigned char* p, int lane, f32x4* S) {
#pragma unroll
    for (int m = 0; m < M; ++m) S[m] = *reinterpret_cast<const f32x4*>(p + m * kBlock + lane * 16);
}
template <int M> __device__ __forceinline__ void store_acc(unsigned char* p, int lane, const f32x4* S) {
#pragma unroll
    for (int m = 0; m < M; ++m) *reinterpret_cast<f32x4*>(p + m * kBlock + lane * 16) = S[m];
}
// ... and as a caller's state holds them
template <int M> __device__ __forceinline__ void load_state(const DeltaOp& a, const float* p, int state, int head, int col, int g, f32x4* S) {
    if (!p || state < 0) {   // uniform over the workgroup
#pragma unroll
        for (int m = 0; m < M; ++m) S[m] = f32x4{0, 0, 0, 0};
        return;
    }
    p += ((long long)state * a.h + head) * a.dk * a.dv;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = row_of(m, 4 * g + e) < a.dk && col < a.dv;
            const unsigned at = unsigned(8 * g * a.dv + col) + unsigned((row_of(m, 0) + e) * a.dv);
            const float v = p[in ? at : 0];
            S[m][e] = in ? v : 0.0f;
        }
}
template <int M> __device__ __forceinline__ void store_state(const DeltaOp& a, float* p, int state, int head, int col, int g, const f32x4* S) {
    if (!p || state < 0) return;
    p += ((long long)state * a.h + head) * a.dk * a.dv;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (row_of(m, 4 * g + e) < a.dk && col < a.dv) p[unsigned(8 * g * a.dv + col) + unsigned((row_of(m, 0) + e) * a.dv)] = S[m][e];
}

// Steps that the scans share.  LDS reads of a step are issued together and fenced; the vector work that comes before the
// products that use them (splitting an operand) covers their latency.
template <int P, int NT, int NK> __device__ __forceinline__ void read_rows(Lds tile, int s, bf16x8 (&f)[NT][P]) {
#pragma unroll
    for (int i = 0; i < NT; ++i) read_frag<P>(tile, NT * NK * kBlock, i * NK + s, f[i]);
}
// block s of a triangular record matrix: by rows of T or A (the record's transpose), row tiles 2 s and on
template <int P, int NT, int MAT> __device__ __forceinline__ void read_lower(Lds mat, int s, bf16x8 (&f)[NT][P]) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
        if ((i >> 1) >= s) read_frag_t<P>(mat, MAT, [&](int y) { return tri_up(y, i >> 1); }, i, s, f[i]);
}
// ... by rows of T^T or A^T, row tiles up to 2 s + 1
template <int P, int NT, int MAT> __device__ __forceinline__ void read_upper(Lds mat, int s, bf16x8 (&f)[NT][P]) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
        if ((i >> 1) <= s) read_frag<P>(mat, MAT, tri_up(i, s), f[i]);
}
// c[i] += f[i] b over the row tiles that block s of a lower / an upper triangular matrix has
template <bool LOWER, int NT, int PA, int PB> __device__ __forceinline__ void mul_tri(int s, const bf16x8 (&f)[NT][PA], const bf16x8 (&b)[PB], f32x4* c) {
    for_pairs<PA, PB>([&](int x, int y) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
            if (LOWER ? (i >> 1) >= s : (i >> 1) <= s) c[i] = mfma(f[i][x], b[y], c[i]);
    });
}
template <int NT, int PA, int PB> __device__ __forceinline__ void mul_tri_t(int s, const bf16x8 (&b)[PB], const bf16x8 (&f)[NT][PA], f32x4* c) {
    for_pairs<PA, PB>([&](int x, int y) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
            if ((i >> 1) >= s) c[i] = mfma(b[y], f[i][x], c[i]);
    });
}
// S[m] += (rows' transpose)[m] b for the contraction blocks of b, GROUP tiles of S at a time, the next group's
// fragments on their way
template <int P, int M, int NK, int NT, int NP> __device__ __forceinline__ void add_outer(Lds tile, const bf16x8 (&b)[NP][MID], f32x4* S) {
    constexpr int GROUP = P == 1 ? 4 : 2;
    bf16x8 f[2][GROUP][P];
    const auto read = [&](int n, int buf) {   // group n of (contraction block, tiles)
#pragma unroll
        for (int x = 0; x < GROUP; ++x) {
            const int m = n % (M / GROUP) * GROUP + x;
            read_frag_t<P>(tile, NT * NK * kBlock, [&](int i) { return i * NK + (m >> 1); }, m, n / (M / GROUP), f[buf][x]);
        }
    };
    constexpr int GROUPS = NP * M / GROUP;
    read(0, 0);
    fence();
#pragma unroll
    for (int n = 0; n < GROUPS; ++n) {
        if (n + 1 < GROUPS) read(n + 1, (n + 1) & 1);
        fence();
        mul(f[n & 1], b[n / (M / GROUP)], S + n % (M / GROUP) * GROUP);
        fence();
    }
}
__device__ __forceinline__ f32x4 read_vec(Lds vec, int at) { return *(LdsVec)(vec + 4 * at); }

// Long sequences with few heads would leave most of the chip idle, so they are cut into segments of `a.segment` chunks
// that scan at the same time.  Over a segment S' = M S + N; delta_transit_kernel finds M (from S = I, v = 0) and N (from
// S = 0) of every segment but a sequence's last, delta_join_kernel the states between the segments, and the scan proper
// begins each segment from its own.  The same M, transposed, carries the gradient of the state backward.
__device__ __forceinline__ long long seg_tokens(const DeltaOp& a, int C) { return a.segment * C; }

// A wave finds 16 columns of N (the first tiles: columns of v) or of M (the others: columns of the identity).  A training
// call needs M of the last segment as well.  At 128 x 128 the 16 tiles go to two workgroups where each has a compute unit
// (3.7 us a step), else to one, where they share K and T (5.4 us a step of both; a second round of the halves 7.4).  In fp16
// the one has 4 registers too few of its 128 and spills them.
template <typename T, int NK, int W, bool TRAIN, bool WHOLE>
__global__ void __launch_bounds__(64 * W) delta_transit_kernel(DeltaOp a) {
    typedef Record<T> R;
    typedef Feed<T, NK, W, WHOLE, false, R::A_AT> Reader;   // T and the vectors: A is not needed
    static_assert(Reader::TWO_X, "one stage of X needs xs_read");
    constexpr int C = R::C, NT = R::NT, NP = R::NP, P = Parts<T>::IN, M = 2 * NK;
    constexpr int COLUMNS = M * NK * MID * kBlock;
    __shared__ __attribute__((aligned(1024))) unsigned char mem[Reader::BYTES > COLUMNS ? Reader::BYTES : COLUMNS];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int vtiles = 2 * ((a.dv + 31) / 32), slices = (vtiles + M + W - 1) / W;
    Item it;
    if (!item_of(a, slots_of(a, seg_tokens(a, C)), a.h, slices, &it)) return;
    const int slice = it.slice, head = it.head;
    const long long slot = it.slot;
    constexpr long long REC = R::BYTES;
    const bool find_m = slice * W + wave >= vtiles, with_v = slice * W < vtiles;   // this wave; any of the workgroup
    Piece p;   // the returns are uniform over the workgroup
    if (!piece_of(a, slot, seg_tokens(a, C), &p) || p.len <= seg_tokens(a, C)) return;
    const bool last = (p.c + 1) * seg_tokens(a, C) >= p.len;
    if (last && !(TRAIN && slice * W + W > vtiles)) return;
    const int hq = head / (a.h / a.hk);
    const int tile = slice * W + wave - (find_m ? vtiles : 0), col = row_of(tile, r);
    const int at = 16 * slot_of(r, g), at_t = 16 * slot_of(4 * g + (r >> 2), r & 3);
    Reader in;
    in.mem = mem;
    in.k = static_cast<const T*>(a.k) + p.begin * a.k_stride + hq * a.k_head;
    in.q = nullptr;
    in.x = static_cast<const T*>(a.v) + p.begin * a.v_stride + head * a.v_head;
    in.rec_stride = a.h * REC;
    in.rec = a.records + (p.begin / C + p.seq) * in.rec_stride + head * REC;
    in.k_stride = a.k_stride;
    in.x_stride = a.v_stride;
    in.len = p.len;
    in.dk = a.dk;
    in.dv = a.dv;
    in.tid = tid;
    in.col = col;
    in.xcol = slice * W * 16;
    f32x4 S[M];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) S[m][e] = find_m && row_of(m, 4 * g + e) == col ? 1.0f : 0.0f;
    const long long chunks = (p.len + C - 1) / C, first = p.c * a.segment;
    const long long end = chunks - first > a.segment ? first + a.segment : chunks;
    in.fetch(first, 0, with_v);
    in.commit(0, true);
    for (long long c = first; c < end; ++c) {
        const int st = int(c - first) & 1;
        const bool more = c + 1 < end;
        in.advance();
        const Lds kt = (Lds)in.k_tile(st), rec = (Lds)in.record(st), vec = rec + R::VEC_AT;
        f32x4 x[NT], v[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) x[i] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NK; ++s) {
            bf16x8 sf[MID], kf[NT][P];
            read_rows<P, NT, NK>(kt + at, s, kf);
            fence();
            split8<MID>(S[2 * s], S[2 * s + 1], sf);
            mul(kf, sf, x);
            if (s < 2 && more) in.fetch_piece(2 * s, c + 1, st ^ 1, with_v);   // K, X
        }
        bf16x8 tf[NT][MID], rf[NP][MID];
        if (find_m) {
#pragma unroll
            for (int i = 0; i < NT; ++i) v[i] = f32x4{0, 0, 0, 0};
        } else {
            in.columns(st, v);
        }
        fence();
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const f32x4 gam = read_vec(vec, row_of(i, 4 * g)), bet = read_vec(vec, 2 * C + row_of(i, 4 * g));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = bet[e] * (v[i][e] - gam[e] * x[i][e]);
        }
#pragma unroll
        for (int s = 0; s < NP; ++s) split8<MID>(x[2 * s], x[2 * s + 1], rf[s]);
#pragma unroll
        for (int i = 0; i < NT; ++i) x[i] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NP; ++s) {
            read_lower<MID, NT, R::MAT>(rec + at_t, s, tf);
            fence();
            mul_tri<true>(s, tf, rf[s], x);
        }
        if (more) in.fetch_piece(3, c + 1, st ^ 1, with_v);   // the record
#pragma unroll
        for (int i = 0; i < NT; ++i) x[i] *= read_vec(vec, C + row_of(i, 4 * g));
#pragma unroll
        for (int s = 0; s < NP; ++s) split8<MID>(x[2 * s], x[2 * s + 1], rf[s]);
        const float all = read_vec(vec, 3 * C)[0];
#pragma unroll
        for (int m = 0; m < M; ++m) S[m] *= all;
        add_outer<P, M, NK, NT>(kt + at_t, rf, S);
        in.commit(st ^ 1, more);
    }
    if (!find_m && !last) store_acc<M>(a.seg_n + ((slot * a.h + head) * vtiles + tile) * M * kBlock, lane, S);
    // M by its rows, [M row tiles][NK], for the join, which takes it as a left operand; for training also by its columns,
    // which are the rows of M^T
    const long long at_slot = (slot * a.h + head) * M * NK * MID * kBlock;
    if (find_m && tile < M) {
#pragma unroll
        for (int s = 0; s < NK; ++s) {
            bf16x8 sf[MID];
            split8<MID>(S[2 * s], S[2 * s + 1], sf);
#pragma unroll
            for (int p = 0; p < MID; ++p) *(LdsFrag)((Lds)mem + ((tile * NK + s) * MID + p) * kBlock + at) = sf[p];
            if (TRAIN) store_frag<MID>(a.seg_mt + at_slot + (tile * NK + s) * MID * kBlock, at, sf);
        }
    }
    __syncthreads();
    // the pairs of columns that this workgroup has (tiles and W are even, so a pair is never split)
    const int begin = slice * W > vtiles ? slice * W - vtiles : 0, end_m = slice * W + W - vtiles < M ? slice * W + W - vtiles : M;
    for (int b = wave; b < M * ((end_m - begin) / 2); b += W) {
        const int m = b % M, s = begin / 2 + b / M;
        bf16x8 f[MID];
        read_frag_t<MID>((Lds)mem + at_t, kBlock, [&](int x) { return (x * NK + (m >> 1)) * MID; }, m, s, f);
        store_frag<MID>(a.seg_m + at_slot + (m * NK + s) * MID * kBlock, at, f);
    }
}

// The states between a sequence's segments, S' = M S + N from the first segment on; BACK: the gradients of the states,
// dS = M^T dS' + N from the last one.  The steps depend on each other, so a step is made short: a workgroup has 16
// columns, each of its NK waves two row tiles of M, which it loads a step ahead as the left operands that they are.  Its
// two tiles of S are one contraction block of the next step, which the waves hand each other through LDS.  1.6 us a step at
// 128 x 128 (45 us for 28 of them): the handing over and M from L2, 96 KB a step, not the products (0.4 us).
template <typename T, int NK, bool BACK>
__global__ void __launch_bounds__(64 * NK) delta_join_kernel(DeltaOp a, const float* from) {
    constexpr int C = Parts<T>::C, M = 2 * NK;
    __shared__ __attribute__((aligned(1024))) unsigned char mem[2 * NK * MID * kBlock];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int vtiles = 2 * ((a.dv + 31) / 32);
    Item it;
    if (!item_of(a, a.n_seqs, a.h, vtiles, &it)) return;   // uniform
    const int tile = it.slice, head = it.head, seq = int(it.slot);
    const long long begin = seq_begin(a, seq), len = seq_len(a, seq, begin), size = seg_tokens(a, C);
    const long long segs = (len + size - 1) / size, slot0 = begin / size + seq;
    if (segs < 2) return;   // uniform
    const int at = 16 * slot_of(r, g);
    // step j applies the transition of segment j (BACK: of segment segs - 1 - j) and leaves what the next one starts from
    const auto seg = [&](long long j) { return slot0 + (BACK ? segs - 1 - j : j); };
    struct Left {   // this wave's two row tiles of a transition and its two tiles of N
        bf16x8 m[2][NK][MID];
        f32x4 n[2];
    };
    const auto load = [&](long long j, Left& x) {
        if (j + 1 >= segs) return;
        const unsigned char* m = (BACK ? a.seg_mt : a.seg_m) + ((seg(j) * a.h + head) * M + 2 * wave) * (long long)(NK * MID * kBlock) + at;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int s = 0; s < NK; ++s)
#pragma unroll
                for (int p = 0; p < MID; ++p) x.m[y][s][p] = *reinterpret_cast<const bf16x8*>(m + ((y * NK + s) * MID + p) * kBlock);
        load_acc<2>(a.seg_n + (((seg(j) * a.h + head) * vtiles + tile) * M + 2 * wave) * (long long)kBlock, lane, x.n);
    };
    f32x4 S[2], all[M];
    load_state<M>(a, from, state_of(a, seq), head, row_of(tile, r), g, all);
#pragma unroll
    for (int m = 0; m < M; ++m)
        if (m >> 1 == wave) S[m & 1] = all[m];
    const auto step = [&](long long j, Left& x) {
        const Lds to = (Lds)mem + int(j & 1) * (NK * MID * kBlock);   // the stage that no wave reads any more
        bf16x8 own[MID];
        split8<MID>(S[0], S[1], own);
#pragma unroll
        for (int p = 0; p < MID; ++p) *(LdsFrag)(to + (wave * MID + p) * kBlock + lane * 16) = own[p];
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // LDS alone: the loads ahead stay in flight
        f32x4 acc[4] = {x.n[0], x.n[1], {0, 0, 0, 0}, {0, 0, 0, 0}};      // even and odd contraction blocks apart
#pragma unroll
        for (int s = 0; s < NK; s += 2) {
            bf16x8 sf[2][MID];
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int p = 0; p < MID; ++p) sf[y][p] = *(LdsFrag)(to + ((s + y) * MID + p) * kBlock + lane * 16);
            for_pairs<MID, MID>([&](int p, int q) {
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int z = 0; z < 2; ++z) acc[2 * y + z] = mfma(x.m[z][s + y][p], sf[y][q], acc[2 * y + z]);
            });
        }
        load(j + 2, x);
        S[0] = acc[0] + acc[2];
        S[1] = acc[1] + acc[3];
        store_acc<2>(a.seg_s + (((seg(j) + (BACK ? -1 : 1)) * a.h + head) * vtiles + tile) * (long long)(M * kBlock) + 2 * wave * kBlock, lane, S);
    };
    if (!BACK)   // the first segment too begins from here: the last one may have stored over state_in before it starts
        store_acc<2>(a.seg_s + ((slot0 * a.h + head) * vtiles + tile) * (long long)(M * kBlock) + 2 * wave * kBlock, lane, S);
    Left even, odd;   // two steps in flight
    load(0, even);
    load(1, odd);
    for (long long j = 0; j + 1 < segs; j += 2) {
        step(j, even);
        if (j + 2 < segs) step(j + 1, odd);
    }
}

// W waves, 16 columns of v each, over one segment.  At 128 x 128 in bf16 a step of 64 tokens takes 4.6 us with four waves, and
// 5 to 6 with eight (232 segments of 9 steps: 77 us).  No unit is busy half of that: the matrix cores 32 %, the vector units
// 32 %, LDS some 40 % (690 KB a step at 128 bytes a clock: every wave reads K, Q, T and A for its 16 columns); 162 MB read
// and 34 written are 2.5 TB/s.  A step is a chain -- K S, R, T R, A U, S -- whose links wait for each other inside a wave, and the one or two
// waves of a SIMD hide too little of it.  Two more, at 128 registers, change nothing (fp32 x 64 keys, 128 sequences of 321
// tokens x 6 heads: 164 us against 163).  General loads of two-byte types with 128 keys spill 5 registers of 256.
template <typename T, int NK, int W, bool TRAIN, bool WHOLE>
__global__ void __launch_bounds__(64 * W) delta_scan_kernel(DeltaOp a) {
    typedef Record<T> R;
    constexpr int C = R::C, NT = R::NT, NP = R::NP, P = Parts<T>::IN, M = 2 * NK;
    typedef Feed<T, NK, W, WHOLE, true, R::BYTES> Reader;
    constexpr long long REC = R::BYTES;
    __shared__ __attribute__((aligned(1024))) unsigned char mem[Reader::BYTES];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slices = (a.dv + 16 * W - 1) / (16 * W);
    Item it;
    Piece p;   // the returns are uniform over the workgroup
    if (!item_of(a, slots_of(a, seg_tokens(a, C)), a.h, slices, &it) || !piece_of(a, it.slot, seg_tokens(a, C), &p)) return;
    const int slice = it.slice, head = it.head;
    const long long slot = it.slot;
    const int hq = head / (a.h / a.hk), tile = slice * W + wave, col = row_of(tile, r);   // this lane's column of v
    const int vtiles = 2 * ((a.dv + 31) / 32);
    const long long chunks = (p.len + C - 1) / C, slot0 = p.begin / C + p.seq;
    const long long first = p.c * a.segment, end = chunks - first > a.segment ? first + a.segment : chunks;
    const int at = 16 * slot_of(r, g), at_t = 16 * slot_of(4 * g + (r >> 2), r & 3);
    Reader in;
    in.mem = mem;
    in.k = static_cast<const T*>(a.k) + p.begin * a.k_stride + hq * a.k_head;
    in.q = static_cast<const T*>(a.q) + p.begin * a.q_stride + hq * a.q_head;
    in.x = static_cast<const T*>(a.v) + p.begin * a.v_stride + head * a.v_head;
    in.rec_stride = a.h * REC;
    in.rec = a.records + slot0 * in.rec_stride + head * REC;
    in.k_stride = a.k_stride;
    in.q_stride = a.q_stride;
    in.x_stride = a.v_stride;
    in.len = p.len;
    in.dk = a.dk;
    in.dv = a.dv;
    in.tid = tid;
    in.col = col;
    in.xcol = slice * W * 16;
    if (first < end) in.fetch(first, 0, true);
    f32x4 S[M];
    const int state = state_of(a, p.seq);
    if (p.len <= seg_tokens(a, C)) load_state<M>(a, a.state_in, state, head, col, g, S);
    else load_acc<M>(a.seg_s + ((slot * a.h + head) * vtiles + (tile < vtiles ? tile : 0)) * M * kBlock, lane, S);
    in.commit(0, first < end);

    // a chunk's o waits in registers until the next step has begun: a step's end does not wait for its stores
    typename Loose4<T>::type held[NT];
    const int c0 = row_of(tile, 4 * g);
    const auto release = [&](long long c) {
        const long long left = p.len - c * C;
        const int valid = left < C ? int(left) : C;
        T* op = static_cast<T*>(a.o) + (p.begin + c * C) * a.o_stride + head * a.o_head + c0;
        const bool cols = WHOLE || c0 + 4 <= a.dv;
        if (c0 >= a.dv) return;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int t = row_of(i, r);
            if (t >= valid) continue;
            T* to = WHOLE ? op + unsigned(t) * unsigned(a.o_stride) : op + t * a.o_stride;
            if (cols) {
                *reinterpret_cast<typename Loose4<T>::type*>(to) = held[i];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c0 + e < a.dv) to[e] = held[i][e];
            }
        }
    };
    for (long long c = first; c < end; ++c) {
        const int st = int(c - first) & 1;
        const long long next = c + 1 < end ? c + 1 : c;   // the last step fetches its own chunk again, to no use
        in.advance();
        if (c > first) release(c - 1);
        const Lds kt = (Lds)in.k_tile(st), qt = (Lds)in.q_tile(st), rec = (Lds)in.record(st), vec = rec + R::VEC_AT;
        f32x4 x[NT], o[NT], v[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) x[i] = o[i] = f32x4{0, 0, 0, 0};
        // K S, the next block of S split while the products of one run
        bf16x8 sf[NK][MID], kf[2][NT][P];
        s16x4 xs[NT];
        if constexpr (!Reader::TWO_X) in.read_x(st, xs);   // here the waves are still together, so the barrier costs least
        read_rows<P, NT, NK>(kt + at, 0, kf[0]);
        split8<MID>(S[0], S[1], sf[0]);
        fence();
        in.xs_read();
#pragma unroll
        for (int s = 0; s < NK; ++s) {
            if (s + 1 < NK) {
                read_rows<P, NT, NK>(kt + at, s + 1, kf[(s + 1) & 1]);
                split8<MID>(S[2 * s + 2], S[2 * s + 3], sf[s + 1]);
            }
            mul(kf[s & 1], sf[s], x);
            interleave<NT * (P == 1 ? 3 : P == 2 ? 5 : 6), 4, NT * P>();
            fence();
        }
        if (TRAIN && tile < vtiles) store_acc<M>(a.starts + (((slot0 + c) * a.h + head) * vtiles + tile) * M * kBlock, lane, S);
        in.fetch_piece(0, next, st ^ 1, true);   // K
        // R while (Q S)^T runs: the same fragments with the operands' places exchanged, so that a lane ends up with four
        // columns of one token and stores them at once
        bf16x8 tf[NT][MID], rf[NP][MID], qf[2][NT][P];
        read_rows<P, NT, NK>(qt + at, 0, qf[0]);
        if constexpr (Reader::TWO_X) in.read_x(st, xs);
        in.widen(xs, v);
        f32x4 gam[NT], bet[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            gam[i] = read_vec(vec, row_of(i, 4 * g));
            bet[i] = read_vec(vec, 2 * C + row_of(i, 4 * g));
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = bet[i][e] * (v[i][e] - gam[i][e] * x[i][e]);
#pragma unroll
        for (int s = 0; s < NP; ++s) split8<MID>(x[2 * s], x[2 * s + 1], rf[s]);
#pragma unroll
        for (int s = 0; s < NK; ++s) {
            if (s + 1 < NK) read_rows<P, NT, NK>(qt + at, s + 1, qf[(s + 1) & 1]);
            mul_t(sf[s], qf[s & 1], o);
        }
        fence();
        in.fetch_piece(1, next, st ^ 1, true);   // Q
        read_lower<MID, NT, R::MAT>(rec + at_t, 0, tf);
        bf16x8 af[NT][MID];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            x[i] = f32x4{0, 0, 0, 0};
            o[i] *= a.scale * *(__attribute__((address_space(3))) float*)(vec + 4 * row_of(i, r));
        }
#pragma unroll
        for (int s = 0; s < NP; ++s) {
            if (s) read_lower<MID, NT, R::MAT>(rec + at_t, s, tf);
            mul_tri<true>(s, tf, rf[s], x);
        }
        fence();
        in.fetch_piece(2, next, st ^ 1, true);   // X
        in.fetch_piece(3, next, st ^ 1, true);   // the record
        read_lower<MID, NT, R::MAT>(rec + R::A_AT + at_t, 0, af);
        fence();
#pragma unroll
        for (int s = 0; s < NP; ++s) split8<MID>(x[2 * s], x[2 * s + 1], rf[s]);   // U
        if (TRAIN && tile < vtiles) store_acc<NT>(a.u + (((slot0 + c) * a.h + head) * vtiles + tile) * NT * kBlock, lane, x);
        fence();
        // S = exp(G_C) S + K^T (exp(G_C - G) U), split while A U runs
        bf16x8 lf[NP][MID];
#pragma unroll
        for (int i = 0; i < NT; ++i) x[i] *= read_vec(vec, C + row_of(i, 4 * g));
#pragma unroll
        for (int s = 0; s < NP; ++s) split8<MID>(x[2 * s], x[2 * s + 1], lf[s]);
        const float all = read_vec(vec, 3 * C)[0];
#pragma unroll
        for (int m = 0; m < M; ++m) S[m] *= all;
#pragma unroll
        for (int s = 0; s < NP; ++s) {
            if (s) read_lower<MID, NT, R::MAT>(rec + R::A_AT + at_t, s, af);
            mul_tri_t(s, rf[s], af, o);
        }
        interleave<R::BLOCKS * 6, 6>();
        fence();
        add_outer<P, M, NK, NT>(kt + at_t, lf, S);
#pragma unroll
        for (int i = 0; i < NT; ++i) held[i] = __builtin_convertvector(o[i], typename Loose4<T>::type);
        in.commit(st ^ 1, c + 1 < end);
    }
    if (first < end) release(end - 1);
    if (end == chunks) store_state<M>(a, a.state_out, state, head, col, g, S);
}

// ------------------------------------------------------------------------------------------ token by token
// Few tokens a sequence: the recurrence itself in fp32, a wave per 32 columns of a head's state.  Lane (rg, cg) holds
// rows rg NR .. rg NR + NR - 1 of columns 4 cg .. 4 cg + 3; S^T k and S^T q are taken on the state before the token in
// one pass over it, o = c (a S^T q + (k . q) u).  Bound by the states' bytes: one token of 192 sequences x 16 heads x 128 x
// 128 moves 405 MB in 79 us, 5.1 TB/s, a large copy's rate.
template <typename T, int NR>
__global__ void __launch_bounds__(256) delta_token_kernel(DeltaOp a) {
    const int slices = (a.dv + 31) / 32;
    const long long item = blockIdx.x * 4LL + (threadIdx.x >> 6);
    if (item >= (long long)a.n_seqs * a.h * slices) return;
    const int lane = threadIdx.x & 63, cg = lane & 7, rg = lane >> 3;
    const int slice = int(item % slices), head = int(item / slices % a.h), seq = int(item / slices / a.h);
    const int hq = head / (a.h / a.hk), c0 = slice * 32 + 4 * cg, x0 = rg * NR;
    const long long begin = seq_begin(a, seq), len = seq_len(a, seq, begin);
    const int state = state_of(a, seq);
    const int rows = a.dk - x0 < NR ? a.dk - x0 : NR;          // may be 0 or less
    const bool whole = c0 + 4 <= a.dv;
    f32x4 S[NR];
    typedef Loose4<float>::type Quad;
#pragma unroll
    for (int j = 0; j < NR; ++j) {
        S[j] = f32x4{0, 0, 0, 0};
        if (a.state_in && state >= 0 && j < rows && c0 < a.dv) {
            const float* p = a.state_in + (((long long)state * a.h + head) * a.dk + x0 + j) * a.dv + c0;
            if (whole) S[j] = *reinterpret_cast<const Quad*>(p);
            else
                for (int e = 0; e < 4; ++e) S[j][e] = c0 + e < a.dv ? p[e] : 0.0f;
        }
    }
    struct Token {   // as stored
        typename Loose8<T>::type k[NR / 8], q[NR / 8];
        T v[4];
        float g, beta;
    } next;
    const auto fetch = [&](long long t) {
        const T* kp = static_cast<const T*>(a.k) + t * a.k_stride + hq * a.k_head + x0;
        const T* qp = static_cast<const T*>(a.q) + t * a.q_stride + hq * a.q_head + x0;
        const T* vp = static_cast<const T*>(a.v) + t * a.v_stride + head * a.v_head + c0;
#pragma unroll
        for (int j = 0; j < NR / 8; ++j) {
            next.k[j] = load8(kp, 8 * j, rows);
            next.q[j] = load8(qp, 8 * j, rows);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) next.v[e] = c0 + e < a.dv ? vp[e] : T(0.0f);
        next.g = a.g[t * a.g_stride + head];
        next.beta = a.beta[t * a.beta_stride + head];
    };
    if (len > 0) fetch(begin);
    for (long long t = begin; t < begin + len; ++t) {
        float k[NR], q[NR], v[4];
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            k[j] = float(next.k[j / 8][j % 8]);
            q[j] = float(next.q[j / 8][j % 8]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = float(next.v[e]);
        const float dec = expf(next.g), bet = next.beta;
        if (t + 1 < begin + len) fetch(t + 1);
        float sum[9] = {};   // S^T k, S^T q, k . q
#pragma unroll
        for (int j = 0; j < NR; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum[e] = __builtin_fmaf(k[j], S[j][e], sum[e]);
                sum[4 + e] = __builtin_fmaf(q[j], S[j][e], sum[4 + e]);
            }
            sum[8] = __builtin_fmaf(k[j], q[j], sum[8]);
        }
#pragma unroll
        for (int e = 0; e < 9; ++e) {   // over the row groups, lanes 8, 16 and 32 across
            sum[e] += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, sum[e]), 0x128, 0xf, 0xf, false));
            sum[e] = across32(across16(sum[e]));
        }
        float u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = bet * (v[e] - dec * sum[e]);
#pragma unroll
        for (int j = 0; j < NR; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[j][e] = __builtin_fmaf(k[j], u[e], dec * S[j][e]);
        if (rg == 0) {
            T* op = static_cast<T*>(a.o) + t * a.o_stride + head * a.o_head + c0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c0 + e < a.dv) op[e] = T(a.scale * (dec * sum[4 + e] + sum[8] * u[e]));
        }
    }
    if (a.state_out && state >= 0 && c0 < a.dv)
#pragma unroll
        for (int j = 0; j < NR; ++j)
            if (j < rows) {
                float* p = a.state_out + (((long long)state * a.h + head) * a.dk + x0 + j) * a.dv + c0;
                if (whole) *reinterpret_cast<Quad*>(p) = S[j];
                else
                    for (int e = 0; e < 4; ++e)
                        if (c0 + e < a.dv) p[e] = S[j][e];
            }
}

// ------------------------------------------------------------------------------------------ gradients
// With dS' the gradient of the state after a chunk and R = diag(b) (V - diag(exp G) K S), so that U = T R:
//
//   dU = A^T dO + diag(exp(G_C - G)) K dS',   dR = T^T dU,   dV = diag(b) dR
//   dS = exp(G_C) dS' + c Q^T diag(exp G) dO - K^T diag(b exp G) dR
//
// is a scan like the forward one, last chunk first, and leaves dS' and dR of every chunk, again as fragments.  What is
// left mixes no chunks (delta_grad_kernel).  With X1 = dO S^T, X2 = dR S^T, X3 = U dS'^T, D as above, and the lower
// triangular dA = c D (dO U^T), M = -D (dR U^T) (M without its diagonal):
//
//   dq_i = c exp(G_i) X1_i + (dA K)_i
//   k as it reads the state:   kr_i = b_i ((M K)_i - exp(G_i) X2_i)
//   k as it is written to it:  kw_i = (M^T diag(b) K)_i + (dA^T Q)_i + exp(G_C - G_i) X3_i
//   dk = kr + kw,   db_i = dR_i . v_i + k_i . ((M K)_i - exp(G_i) X2_i)
//
// G enters as q_i exp(G_i), as k_i exp(G_i) where it reads and as k_i exp(-G_i) where it is written, so its gradient is
// q_i . dq_i + k_i . (kr_i - kw_i), plus dS' . S' at the chunk's end, and g's is the sum of G's over the tokens from its
// own to the chunk's end.  Terms that this would add and take away again are left out: dA's diagonal, and the part of kw
// that reaches S', of which the tokens before g's own remain.
// FIND: the gradient that a segment hands to the one before it when none reaches its own end (N of delta_join_kernel).
// Bound as the scan is: 128 segments of 8 chunks x 128 x 128 in bf16 take 60 us, to FIND 45.
template <typename T, int NK, int W, bool FIND, bool WHOLE>
__global__ void __launch_bounds__(64 * W) delta_back_kernel(DeltaOp a, DeltaGrad d) {
    typedef Record<T> R;
    constexpr int C = R::C, NT = R::NT, NP = R::NP, P = Parts<T>::IN, M = 2 * NK;
    typedef Feed<T, NK, W, WHOLE, true, R::BYTES> Reader;
    static_assert(Reader::TWO_X, "one stage of X needs xs_read");
    __shared__ __attribute__((aligned(1024))) unsigned char mem[Reader::BYTES];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slices = (a.dv + 16 * W - 1) / (16 * W);
    Item it;
    Piece p;   // the returns are uniform over the workgroup
    if (!item_of(a, slots_of(a, seg_tokens(a, C)), a.h, slices, &it) || !piece_of(a, it.slot, seg_tokens(a, C), &p)) return;
    if (FIND && p.c == 0) return;
    const int slice = it.slice, head = it.head;
    const long long slot = it.slot;
    const int hq = head / (a.h / a.hk), tile = slice * W + wave, col = row_of(tile, r);
    const int vtiles = 2 * ((a.dv + 31) / 32);
    const long long chunks = (p.len + C - 1) / C, slot0 = p.begin / C + p.seq;
    const long long first = p.c * a.segment, end = chunks - first > a.segment ? first + a.segment : chunks;
    const int at = 16 * slot_of(r, g), at_t = 16 * slot_of(4 * g + (r >> 2), r & 3);
    Reader in;
    in.mem = mem;
    in.k = static_cast<const T*>(a.k) + p.begin * a.k_stride + hq * a.k_head;
    in.q = static_cast<const T*>(a.q) + p.begin * a.q_stride + hq * a.q_head;
    in.x = static_cast<const T*>(d.d_o) + (p.begin * a.h + head) * a.dv;
    in.rec_stride = a.h * (long long)R::BYTES;
    in.rec = a.records + slot0 * in.rec_stride + head * (long long)R::BYTES;
    in.k_stride = a.k_stride;
    in.q_stride = a.q_stride;
    in.x_stride = (long long)a.h * a.dv;
    in.len = p.len;
    in.dk = a.dk;
    in.dv = a.dv;
    in.tid = tid;
    in.col = col;
    in.xcol = slice * W * 16;
    if (first < end) in.fetch(end - 1, 0, true);
    f32x4 S[M];   // dS
    const int state = state_of(a, p.seq);
    if (FIND) {
#pragma unroll
        for (int m = 0; m < M; ++m) S[m] = f32x4{0, 0, 0, 0};
    } else if (end == chunks) {
        load_state<M>(a, d.d_state_out, state, head, col, g, S);
    } else {
        load_acc<M>(a.seg_s + ((slot * a.h + head) * vtiles + (tile < vtiles ? tile : 0)) * M * kBlock, lane, S);
    }
    in.commit(0, first < end);
    for (long long c = end - 1; c >= first; --c) {
        const int st = int(end - 1 - c) & 1;
        const int valid = p.len - c * C < C ? int(p.len - c * C) : C;
        const bool more = c > first;
        in.advance();
        const Lds kt = (Lds)in.k_tile(st), qt = (Lds)in.q_tile(st), rec = (Lds)in.record(st), vec = rec + R::VEC_AT;
        const long long at_slot = ((slot0 + c) * a.h + head) * vtiles + tile;
        if (!FIND && tile < vtiles) store_acc<M>(d.ends + at_slot * M * kBlock, lane, S);
        f32x4 o[NT], u[NT];   // dO, dU
        in.columns(st, o);
#pragma unroll
        for (int i = 0; i < NT; ++i) u[i] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NK; ++s) {
            bf16x8 sf[MID], kf[NT][P];
            read_rows<P, NT, NK>(kt + at, s, kf);
            fence();
            split8<MID>(S[2 * s], S[2 * s + 1], sf);
            mul(kf, sf, u);
            if (s < 2 && more) in.fetch_piece(s, c - 1, st ^ 1, true);   // K, Q
        }
        bf16x8 of[NP][P], rf[NP][MID], tf[NT][MID];
        read_upper<MID, NT, R::MAT>(rec + R::A_AT + at, 0, tf);
        fence();
#pragma unroll
        for (int s = 0; s < NP; ++s) split8<P>(o[2 * s], o[2 * s + 1], of[s]);
#pragma unroll
        for (int i = 0; i < NT; ++i) u[i] *= read_vec(vec, C + row_of(i, 4 * g));
#pragma unroll
        for (int s = 0; s < NP; ++s) {
            if (s) read_upper<MID, NT, R::MAT>(rec + R::A_AT + at, s, tf);
            mul_tri<false>(s, tf, of[s], u);
        }
        if (more) {
            in.fetch_piece(2, c - 1, st ^ 1, true);   // X
            in.fetch_piece(3, c - 1, st ^ 1, true);   // the record
        }
        read_upper<MID, NT, R::MAT>(rec + at, 0, tf);
        fence();
#pragma unroll
        for (int s = 0; s < NP; ++s) split8<MID>(u[2 * s], u[2 * s + 1], rf[s]);
#pragma unroll
        for (int i = 0; i < NT; ++i) u[i] = f32x4{0, 0, 0, 0};   // dR
#pragma unroll
        for (int s = 0; s < NP; ++s) {
            if (s) read_upper<MID, NT, R::MAT>(rec + at, s, tf);
            mul_tri<false>(s, tf, rf[s], u);
        }
        if (!FIND && tile < vtiles) store_acc<NT>(d.dr + at_slot * NT * kBlock, lane, u);
        T* vp = static_cast<T*>(d.d_v) + ((p.begin + c * C) * a.h + head) * a.dv;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const f32x4 gam = read_vec(vec, row_of(i, 4 * g)), bet = read_vec(vec, 2 * C + row_of(i, 4 * g));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = row_of(i, 4 * g + e);
                u[i][e] *= bet[e];
                if (!FIND && t < valid && col < a.dv) vp[unsigned(t) * unsigned(a.h * a.dv) + unsigned(col)] = T(u[i][e]);
                u[i][e] *= -gam[e];
                o[i][e] *= a.scale * gam[e];
            }
        }
        bf16x8 gf[NP][MID];
#pragma unroll
        for (int s = 0; s < NP; ++s) {
            split8<MID>(u[2 * s], u[2 * s + 1], rf[s]);
            split8<MID>(o[2 * s], o[2 * s + 1], gf[s]);
        }
        const float all = read_vec(vec, 3 * C)[0];
#pragma unroll
        for (int m = 0; m < M; ++m) S[m] *= all;
        add_outer<P, M, NK, NT>(qt + at_t, gf, S);
        add_outer<P, M, NK, NT>(kt + at_t, rf, S);
        in.commit(st ^ 1, more);
    }
    if (FIND) {
        if (tile < vtiles) store_acc<M>(a.seg_n + ((slot * a.h + head) * vtiles + tile) * M * kBlock, lane, S);
    } else if (p.c == 0) {
        store_state<M>(a, d.d_state_in, state, head, col, g, S);
    }
}

// Eight waves per (chunk, q / k head), one value head of its group after the other: wave (i, part) has token tile i and a
// share of the dk tiles, every product transposed so that a lane holds four key dimensions of one token.  U, dR, S and
// dS' come in as fp32 accumulators, SLAB tiles of v at a time, and are split on the way to LDS: as fp32 they are two
// thirds of what their parts would be, and this kernel and the scans that feed it move more of them than anything else.
// 128 chunks x 4 q / k heads x 2 heads x 128 x 128 in bf16 take 126 us: 285 MB read, 50 written, the matrix cores 11 % and
// the vector units 16 % busy (fp16 x 64 keys, 32 sequences of 321 tokens x 6 heads: 108 us, 14 % and 29 %).  Its phases wait
// for each other at barriers with one workgroup on a compute unit.  With 128 keys the accumulators leave too few registers
// even so: 28 of 256 are spilled in the two-byte types, and sixteen waves, of 128, took 210 us.
template <typename T, int NK, bool WHOLE>
__global__ void __launch_bounds__(512) delta_grad_kernel(DeltaOp a, DeltaGrad d) {
    typedef Record<T> R;
    typedef RowTile<T, NK, 512> Tile;
    constexpr int C = R::C, NT = R::NT, NP = R::NP, P = Parts<T>::IN, M = 2 * NK;
    constexpr int PARTS = 8 / NT, MW = M / PARTS, SLAB = P == 2 && NK == 4 ? 2 : 4;   // v tiles in LDS at a time
    constexpr int U_BYTES = SLAB * NP * MID * kBlock, S_BYTES = SLAB * NK * MID * kBlock, MAT = MID * R::MAT;
    constexpr int FIRST = 2 * U_BYTES + S_BYTES, SECOND = 3 * MAT, REGION = FIRST > SECOND ? FIRST : SECOND;
    constexpr int UU = (SLAB * NP + 7) / 8, SU = SLAB * NK / 8;   // 16 x 32 pieces of U (and dR), of S (and dS') per wave
    __shared__ __attribute__((aligned(1024))) unsigned char mem[REGION + 2 * Tile::BYTES];
    __shared__ double gsum[C];
    __shared__ float vecs[2][3 * C + 1], red[PARTS][3][C], vdot[C], diag[C], ends[8];
    int seq, valid;
    long long begin;
    Item it;
    if (!item_of(a, slots_of(a, C), a.hk, 1, &it) || !chunk_of<C>(a, it.slot, &seq, &begin, &valid)) return;   // uniform
    const int hq = it.head, group = a.h / a.hk;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = wave % NT, part = wave / NT;
    const int at = 16 * slot_of(r, g), at_t = 16 * slot_of(4 * g + (r >> 2), r & 3);
    const int vtiles = 2 * ((a.dv + 31) / 32), token = row_of(i, r);
    const Lds ut = (Lds)mem, rt = ut + U_BYTES, st = rt + U_BYTES, mats = ut, kt = ut + REGION, qt = kt + Tile::BYTES;
    f32x4 dq[MW], dk[MW];
#pragma unroll
    for (int m = 0; m < MW; ++m) dq[m] = dk[m] = f32x4{0, 0, 0, 0};
    // piece n of this wave of a [tiles][BLOCKS] matrix of accumulators: 8 rows of a column per lane, two tiles of it
    const auto load_piece = [&](const unsigned char* p, int b, f32x4 (&v)[2]) {
        v[0] = *reinterpret_cast<const f32x4*>(p + (2 * b) * kBlock + lane * 16);
        v[1] = *reinterpret_cast<const f32x4*>(p + (2 * b + 1) * kBlock + lane * 16);
    };
    const auto put_piece = [&](Lds to, int b, const f32x4 (&v)[2]) {
        bf16x8 f[MID];
        split8<MID>(v[0], v[1], f);
#pragma unroll
        for (int p = 0; p < MID; ++p) *(LdsFrag)(to + (b * MID + p) * kBlock + at) = f[p];
    };

    f32x4 un[UU][2], rn[UU][2], sn[SU][2], en[SU][2];
    const auto fetch = [&](int head, int slab) {   // this wave's pieces of U, dR and S
        const long long at_slot = (it.slot * a.h + head) * vtiles;
        const int tiles = vtiles - slab < SLAB ? vtiles - slab : SLAB;
        const unsigned char *up = a.u + (at_slot + slab) * NT * kBlock, *rp = d.dr + (at_slot + slab) * NT * kBlock;
        const unsigned char* sp = a.starts + (at_slot + slab) * M * kBlock;
#pragma unroll
        for (int n = 0; n < UU; ++n)
            if (wave + 8 * n < tiles * NP) {
                load_piece(up, wave + 8 * n, un[n]);
                load_piece(rp, wave + 8 * n, rn[n]);
            }
#pragma unroll
        for (int n = 0; n < SU; ++n)
            if (wave + 8 * n < tiles * NK) load_piece(sp, wave + 8 * n, sn[n]);
    };
    float rv = 0.0f, gv = 0.0f;   // the next head's vectors and g
    const auto fetch_head = [&](int head) {
        const float* rec = reinterpret_cast<const float*>(a.records + (it.slot * a.h + head) * R::BYTES + R::VEC_AT);
        if (wave == 0 && lane < valid) gv = a.g[(begin + lane) * a.g_stride + head];
        if (tid < 3 * C + 1) rv = rec[tid];
    };
    fetch(hq * group, 0);
    fetch_head(hq * group);
    {
        Tile k, q;
        k.template load<WHOLE>(static_cast<const T*>(a.k) + begin * a.k_stride + hq * a.k_head, a.k_stride, valid, a.dk, tid);
        q.template load<WHOLE>(static_cast<const T*>(a.q) + begin * a.q_stride + hq * a.q_head, a.q_stride, valid, a.dk, tid);
        k.store(mem + REGION, tid);
        q.store(mem + REGION + Tile::BYTES, tid);
    }
    for (int head = hq * group; head < (hq + 1) * group; ++head) {
        const long long at_slot = (it.slot * a.h + head) * vtiles;
        float* vec = vecs[(head - hq * group) & 1];   // two, since the first wave ends a head while the others go on
        if (tid < 3 * C + 1) vec[tid] = rv;
        const float g_token = gv;
        f32x4 x1[MW], x2[MW], x3[MW], job[NT];
        float dot = 0.0f, end = 0.0f;
#pragma unroll
        for (int m = 0; m < MW; ++m) x1[m] = x2[m] = x3[m] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < NT; ++j) job[j] = f32x4{0, 0, 0, 0};
        const T* op = static_cast<const T*>(d.d_o) + ((begin + token) * a.h + head) * a.dv;
        const T* vp = static_cast<const T*>(a.v) + (begin + token) * a.v_stride + head * a.v_head;
        for (int slab = 0; slab < vtiles; slab += SLAB) {
            const int tiles = vtiles - slab < SLAB ? vtiles - slab : SLAB;
            typename Loose8<T>::type ov[SLAB / 2], vv[SLAB / 2];
#pragma unroll
            for (int kb = 0; kb < SLAB / 2; ++kb) {
                const int c0 = 16 * slab + 32 * kb + 8 * g;
                const bool in = token < valid && c0 < a.dv;
                ov[kb] = load8(in ? op : static_cast<const T*>(d.d_o), in ? c0 : 0, in ? a.dv : 0);
                if (part == 0) vv[kb] = load8(in ? vp : static_cast<const T*>(a.v), in ? c0 : 0, in ? a.dv : 0);
            }
#pragma unroll
            for (int n = 0; n < UU; ++n)
                if (wave + 8 * n < tiles * NP) {
                    put_piece(ut, wave + 8 * n, un[n]);
                    put_piece(rt, wave + 8 * n, rn[n]);
                }
            const unsigned char* ep = d.ends + (at_slot + slab) * M * kBlock;
#pragma unroll
            for (int n = 0; n < SU; ++n)
                if (wave + 8 * n < tiles * NK) {
                    put_piece(st, wave + 8 * n, sn[n]);
                    load_piece(ep, wave + 8 * n, en[n]);
                }
            __syncthreads();
#pragma unroll
            for (int kb = 0; kb < SLAB / 2; ++kb) {
                if (kb >= tiles / 2) break;
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = float(ov[kb][e]);
                bf16x8 of[P], rf[MID];
                const auto u_blk = [&](int row_pair) { return [=](int n) { return (n * NP + row_pair) * MID; }; };
                read_frag_t<MID>(rt + at_t, kBlock, u_blk(i >> 1), i, kb, rf);
                split8<P>(y, of);
                if (part == 0) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float x = 0.0f;
#pragma unroll
                        for (int p = MID - 1; p >= 0; --p) x += float(rf[p][e]);
                        dot = __builtin_fmaf(x, float(vv[kb][e]), dot);
                    }
                }
#pragma unroll
                for (int n = 0; n < MW; ++n) {
                    const int m = part * MW + n;
                    bf16x8 sf[1][MID];
                    read_frag_t<MID>(st + at_t, kBlock, [&](int x) { return (x * NK + (m >> 1)) * MID; }, m, kb, sf[0]);
                    mul(sf, rf, x2 + n);
                    mul(sf, of, x1 + n);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if ((j >> 1) > (i >> 1) || j % (PARTS / 2) != part >> 1) continue;
                    bf16x8 uf[1][MID];
                    read_frag_t<MID>(ut + at_t, kBlock, u_blk(j >> 1), j, kb, uf[0]);
                    if (part & 1) mul(uf, rf, job + j);
                    else mul(uf, of, job + j);
                }
            }
            if (slab == 0 && wave == 0) {   // read after the next barriers
                double s = log_decay(g_token);
#pragma unroll
                for (int x = 1; x < C; x *= 2) {
                    const double up = __shfl_up(s, x);
                    if (lane >= x) s += up;
                }
                if (lane < C) gsum[lane] = s;
            }
            __syncthreads();   // S is read: dS' takes its place, its product with S on the way
#pragma unroll
            for (int n = 0; n < SU; ++n)
                if (wave + 8 * n < tiles * NK) {
                    put_piece(st, wave + 8 * n, en[n]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) end = __builtin_fmaf(sn[n][0][e], en[n][0][e], __builtin_fmaf(sn[n][1][e], en[n][1][e], end));
                }
            if (slab + SLAB < vtiles) fetch(head, slab + SLAB);
            else if (head + 1 < (hq + 1) * group) {
                fetch(head + 1, 0);
                fetch_head(head + 1);
            }
            __syncthreads();
            for (int kb = 0; kb < tiles / 2; ++kb) {
                bf16x8 uf[MID];
                read_frag_t<MID>(ut + at_t, kBlock, [&](int n) { return (n * NP + (i >> 1)) * MID; }, i, kb, uf);
#pragma unroll
                for (int n = 0; n < MW; ++n) {
                    const int m = part * MW + n;
                    bf16x8 sf[1][MID];
                    read_frag_t<MID>(st + at_t, kBlock, [&](int x) { return (x * NK + (m >> 1)) * MID; }, m, kb, sf[0]);
                    mul(sf, uf, x3 + n);
                }
            }
            __syncthreads();
        }
        // dA, M and diag(b) M take the place of U, dR and S
        const float gam = vec[token], last = vec[C + token], bet = vec[2 * C + token];
        const double gi = gsum[token];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            if ((j >> 1) > (i >> 1) || j % (PARTS / 2) != part >> 1) continue;
            float x[4], x_own = 0.0f;
            const bool second = part & 1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int jt = row_of(j, 4 * g + e);
                const float dec = decay_of(gi - gsum[jt]);   // past the diagonal it may be anything
                x[e] = jt < token ? (second ? -dec : a.scale * dec) * job[j][e] : 0.0f;
                if (j == i) x_own = (r & 3) == e ? a.scale * job[j][e] : x_own;
            }
            if (!second && j == i && g == r >> 2) diag[token] = x_own;
            const int to = tri(i, j >> 1) * kBlock + at + 8 * (j & 1);
            auto put = [&](Lds mat, float f) {
                typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                f32x4 rest = {f * x[0], f * x[1], f * x[2], f * x[3]};
#pragma unroll
                for (int p = 0; p < MID; ++p) {
                    const bf16x4 h = __builtin_convertvector(rest, bf16x4);
                    *(__attribute__((address_space(3))) bf16x4*)(mat + p * R::MAT + to) = h;
                    rest -= __builtin_convertvector(h, f32x4);
                }
            };
            if (second) {
                put(mats + MAT, 1.0f);
                put(mats + 2 * MAT, bet);
            } else {
                put(mats, 1.0f);
            }
        }
        __syncthreads();
        const float own = diag[token];
        float sg = 0.0f, sb = 0.0f, se = 0.0f;
        const auto cols = [&](int x) { return tri(x, i >> 1); };
        f32x4 kw[MW];   // x1 becomes dq, x2 k's reading part
#pragma unroll
        for (int n = 0; n < MW; ++n) {
            x1[n] *= a.scale * gam;
            x2[n] *= -gam;
            kw[n] = f32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int s = 0; s < NP; ++s) {
            const auto rows = [&](Lds tile, bf16x8 (&f)[MW][P]) {
#pragma unroll
                for (int n = 0; n < MW; ++n) {
                    const int m = part * MW + n;
                    read_frag_t<P>(tile + at_t, NT * NK * kBlock, [&](int x) { return x * NK + (m >> 1); }, m, s, f[n]);
                }
            };
            bf16x8 kf[MW][P], f[MID];
            rows(kt, kf);
            if (s <= i >> 1) {
                read_frag<MID>(mats + at, R::MAT, tri(i, s), f);
                mul(kf, f, x1);
                read_frag<MID>(mats + MAT + at, R::MAT, tri(i, s), f);
                mul(kf, f, x2);
            }
            if (s >= i >> 1) {
                read_frag_t<MID>(mats + 2 * MAT + at_t, R::MAT, cols, i, s, f);
                mul(kf, f, kw);
                rows(qt, kf);
                read_frag_t<MID>(mats + at_t, R::MAT, cols, i, s, f);
                mul(kf, f, kw);
            }
        }
#pragma unroll
        for (int n = 0; n < MW; ++n) {
            const int m = part * MW + n;
            // q and k of this token and these key dimensions, from their tiles (rows past the last token count for nothing)
            float qv[4] = {}, kv[4] = {};
#pragma unroll
            for (int p = P - 1; p >= 0; --p) {
                typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                const int from = (p * NT * NK + i * NK + (m >> 1)) * kBlock + at + 8 * (m & 1);
                const f32x4 q4 = __builtin_convertvector(*(__attribute__((address_space(3))) bf16x4*)(qt + from), f32x4);
                const f32x4 k4 = __builtin_convertvector(*(__attribute__((address_space(3))) bf16x4*)(kt + from), f32x4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    qv[e] += q4[e];
                    kv[e] += k4[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float q1 = x1[n][e], read = x2[n][e], state = last * x3[n][e];
                sg = __builtin_fmaf(qv[e], q1, __builtin_fmaf(kv[e], bet * read - kw[n][e], sg));
                sb = __builtin_fmaf(kv[e], read, sb);
                se = __builtin_fmaf(kv[e], state, se);
                dq[n][e] += __builtin_fmaf(own, kv[e], q1);
                dk[n][e] += __builtin_fmaf(own, qv[e], bet * read + kw[n][e] + state);
            }
        }
        if (token >= valid) sg = sb = se = 0.0f;
#pragma unroll
        for (int x = 16; x < 64; x *= 2) {
            sg += __shfl_xor(sg, x);
            sb += __shfl_xor(sb, x);
            se += __shfl_xor(se, x);
            dot += __shfl_xor(dot, x);
        }
#pragma unroll
        for (int x = 1; x < 64; x *= 2) end += __shfl_xor(end, x);
        if (g == 0) {
            red[part][0][token] = sg;
            red[part][1][token] = sb;
            red[part][2][token] = se;
            if (part == 0) vdot[token] = dot;
        }
        if (lane == 0) ends[wave] = end;
        __syncthreads();
        if (wave == 0) {   // a token per lane: G's gradient, summed from the chunk's end
            double s = 0.0, before = 0.0, all = 0.0;
            float b = 0.0f;
            if (lane < C) {
                b = vdot[lane];
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    s += red[p][0][lane];
                    b += red[p][1][lane];
                    before += red[p][2][lane];
                }
            }
#pragma unroll
            for (int p = 0; p < 8; ++p) all += ends[p];
            const double mine = before;
#pragma unroll
            for (int x = 1; x < C; x *= 2) {
                const double down = __shfl_down(s, x), up = __shfl_up(before, x);
                if (lane + x < C) s += down;
                if (lane >= x) before += up;
            }
            s += before - mine + double(vec[3 * C]) * all;
            if (lane < valid) {
                d.d_g[(begin + lane) * a.h + head] = float(s);
                d.d_beta[(begin + lane) * a.h + head] = b;
            }
        }
    }
    if (token < valid) {
        const long long row = ((begin + token) * a.hk + hq) * a.dk;
#pragma unroll
        for (int n = 0; n < MW; ++n) {
            const int x = row_of(part * MW + n, 4 * g);
            if (x >= a.dk) continue;
            T *qo = static_cast<T*>(d.d_q) + row + x, *ko = static_cast<T*>(d.d_k) + row + x;
            if (x + 4 <= a.dk) {
                *reinterpret_cast<typename Loose4<T>::type*>(qo) = __builtin_convertvector(dq[n], typename Loose4<T>::type);
                *reinterpret_cast<typename Loose4<T>::type*>(ko) = __builtin_convertvector(dk[n], typename Loose4<T>::type);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (x + e < a.dk) {
                        qo[e] = T(dq[n][e]);
                        ko[e] = T(dk[n][e]);
                    }
            }
        }
    }
}

template <class F> void for_type(OpType t, F&& f) {
    if (t == OpType::F32) f(float{});
    else if (t == OpType::F16) f(f16{});
    else f(bf16{});
}
template <class F> void for_keys(int dk, F&& f) {   // 32-wide contraction blocks
    if (dk <= 64) f(std::integral_constant<int, 2>{});
    else f(std::integral_constant<int, 4>{});
}
long long slots_on_host(const DeltaOp& a, long long tokens) { return a.n_tokens / tokens + a.n_seqs; }
unsigned item_grid(long long slots, int heads, int slices) {
    return unsigned((slots * heads * slices + kXcds - 1) / kXcds * kXcds);
}
template <class F> void for_flag(bool on, F&& f) {
    if (on) f(std::true_type{});
    else f(std::false_type{});
}
template <typename T> unsigned scan_grid(const DeltaOp& a, int slices) {
    return item_grid(slots_on_host(a, a.segment * Parts<T>::C), a.h, slices);
}

// Whole, aligned rows: no masks and no partial vectors in the chunk kernels' loads.
bool whole_rows(OpType t, const DeltaOp& a) {
    const long long size = t == OpType::F32 ? 4 : 2, unit = 16 / size;
    const auto fits = [&](const void* p, long long stride, long long head) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % unit == 0 && head % unit == 0 && stride * size * 64 < (1LL << 31);
    };
    return (a.dk == 64 || a.dk == 128) && a.dv % 32 == 0 && fits(a.q, a.q_stride, a.q_head) && fits(a.k, a.k_stride, a.k_head) &&
           fits(a.v, a.v_stride, a.v_head) && fits(a.o, a.o_stride, a.o_head);
}

// at most so many segments of `tokens` each
long long segments_on_host(const DeltaOp& a, long long tokens) {
    return a.offsets ? a.n_tokens / tokens + a.n_seqs : a.n_seqs * ((a.per_seq + tokens - 1) / tokens);
}

// How many chunks a segment has: the count that a model of the kernels' times puts first, or no segments.  The model counts
// steps: in us at 128 x 128, bf16, a start of 15 and 5.2 a step for the scan, 20 and 5.4 for the transitions (12 and 3.7
// where their two halves have a compute unit each), 4 and 1.6 a segment for the join; backward both walks together 45 and
// 7.2 a step, the join 2.6 a segment.  Workgroups that fit into one round of the 256 compute units step together; more of
// them share the units, each with a start worth 3 steps.  (The scan's 5.2 were fitted before its o took the third parts; its
// picks are measured below as they are.)  Where lengths differ the counts are bounds and the end is uneven,
// so there the gain has to be larger.
// Measured, split and whole, in us, calls in a row.  One sequence of 128 x 128: bf16, 8 heads: 512 tokens 42 and 46, 1,024 50
// and 79, 2,048 69 and 151, 16,421 223 and 1,264 (321 tokens stay whole, 37); one head: 512 41 and 47, 16,421 141 and 1,228;
// fp32, 8 heads: 321 tokens 39 and 47, 2,048 79 and 237.  The same steps are counted for fewer keys: fp16, 64 x 128, 8 heads:
// 512 tokens 34 and 45, 4,096 97 and 289; fp32, 64 x 128, 6 heads: 321 tokens 28 and 37.  24 sequences of 1 to 2,500 tokens x
// 16 heads: 250 and 289 (246 in segments one chunk longer); 8 such: 144 and 224 (131 in longer ones); 64 of 1 to 600 x 8
// heads stay whole, 129, against 141 in segments of 12.  With the gradients, bf16, 8 heads: 640 tokens 112 and 134, 2,048
// 163 and 349, 16,421 772 and 2,957 (512 stay whole, 115); 24 packed sequences x 4 heads 315 and 523.
long long segment_of(OpType t, const DeltaOp& a, bool train) {
    const long long whole = 1LL << 40, C = t == OpType::F32 ? 32 : 64;
    const long long longest = !a.offsets ? a.per_seq : a.max_len > 0 && a.max_len < a.n_tokens ? a.max_len : a.n_tokens;
    const long long n = longest > C ? (longest + C - 1) / C : 1;
    const double all = double(a.n_tokens) / double(C);
    const auto steps = [&](double segments, double chunks, long long s) {   // segments and chunks of one head
        const double items = segments * a.h, rounds = double((long long)((items + 255) / 256)) * double(s);
        const double fill = (chunks * a.h + 3 * items) / 256, longer = fill > s ? fill : s, shorter = fill > s ? s : fill;
        return rounds < longer + 0.2 * shorter || items <= 256 ? rounds : longer + 0.2 * shorter;
    };
    const auto segments = [&](long long s) { return double(segments_on_host(a, C * s)); };
    const int halves = a.dv > 64 ? 2 : 1;   // workgroups of four waves backward
    double best = 15 + 5.2 * steps(segments(n), all, n) + (train ? 25 + 4 * steps(halves * segments(n), halves * all, n) : 0);
    long long pick = whole;
    for (long long s = 2; s < n; s += 1 + s / 16) {
        const double m = segments(s), rest = all - 0.5 * double(s) * a.n_seqs;   // a sequence's last segment needs no transition
        double cost = 15 + 5.2 * steps(m, all, s) + 4 + 1.6 * double(n) / double(s);
        cost += m * a.h > 128 ? 20 + 5.4 * steps(m > a.n_seqs ? m - a.n_seqs : 1, rest > 0 ? rest : 0, s) : 12 + 3.7 * double(s);
        if (train) cost += 45 + 7.2 * steps(halves * m, halves * all, s) + 2.6 * double(n) / double(s);
        if (a.offsets) cost *= a.max_len > 0 ? 1.3 : 1.5;   // lengths that differ; a longest one that is not known
        if (cost < best) {
            best = cost;
            pick = s;
        }
    }
    return pick;
}
// Eight waves a workgroup share what they read of K, Q and the records, unless four leave no compute unit without work
// that eight would.  128 segments of 8 chunks x 128 x 128, bf16: 64 us with four, 67 with eight; backward over 192 heads of
// 321 tokens x 64 x 128, fp16: 67 with four, 52 with eight.
bool wide_slices(OpType t, const DeltaOp& a, long long segment) {
    return a.dv > 64 && segments_on_host(a, segment * (t == OpType::F32 ? 32 : 64)) * a.h * 2 > 256;
}

}  // namespace

DeltaSizes delta_sizes(OpType t, const DeltaOp& a, bool train) {
    DeltaSizes s{};
    for_type(t, [&](auto type) {
        typedef decltype(type) T;
        const size_t slots = size_t(slots_on_host(a, Parts<T>::C)) * size_t(a.h), block = size_t(MID) * kBlock;
        const size_t vtiles = 2 * ((size_t(a.dv) + 31) / 32), nk = a.dk <= 64 ? 2 : 4;
        s.records = slots * Record<T>::BYTES;
        if (train) {
            s.starts = slots * vtiles * 2 * nk * kBlock;
            s.u = slots * vtiles * Record<T>::NT * kBlock;
        }
        const long long seg = segment_of(t, a, train) * Parts<T>::C;
        if (seg < a.n_tokens) {
            const size_t segs = size_t(slots_on_host(a, seg)) * size_t(a.h);
            s.seg_m = segs * 2 * nk * nk * block;
            s.seg_n = segs * vtiles * 2 * nk * kBlock;
        }
    });
    return s;
}

// Token by token against chunks, in us.  At 128 x 128 in bf16 one sequence of 16 heads: 6.7 for one token, 10.0 for 4, 19.6 for
// 12, 24 for 16, by chunks 21 for each; 64 such sequences, which fill the chip: 30 for 4 tokens, 61 for 16, 105 for 32, 149 for
// 48, by chunks 107 to 123.  fp16 and fp32 cross in the same places there (12 tokens 19 and 22, 19.6 and 18; 32 tokens 113 and
// 128, 110 and 117).  Smaller heads, whose chunks cost less, cross earlier, which the rule does not follow: 64 sequences x 6
// heads of 64 x 128 in bf16 24 tokens 33 and 34, 32 tokens 42 and 34; x 8 heads of 32 x 32 in fp32 16 tokens 22 and 20, 32
// tokens 38 and 21.
bool delta_by_token(const DeltaOp& a) {
    const long long most = (long long)a.n_seqs * a.h >= 256 ? 32 : 12, longest = a.offsets ? a.max_len : a.per_seq;
    return longest <= most && (!a.offsets || a.max_len > 0);
}

// Whether every launch of a call has fewer than 2^32 threads, HIP's limit; items and workgroups then fit 32 bits by far.
bool delta_launches(OpType t, DeltaOp a, bool train) {
    const auto fits = [](long long groups, int threads) { return (groups + kXcds) * threads < (1LL << 32); };
    if (!train && delta_by_token(a)) return fits(((long long)a.n_seqs * a.h * ((a.dv + 31) / 32) + 3) / 4, 256);
    a.segment = segment_of(t, a, train);
    const long long C = t == OpType::F32 ? 32 : 64, slots = slots_on_host(a, C), segs = slots_on_host(a, C * a.segment);
    const int vtiles = 2 * ((a.dv + 31) / 32), keys = a.dk <= 64 ? 4 : 8, nk = keys / 2;
    const auto sliced = [&](int tiles, int waves) { return fits(segs * a.h * ((tiles + waves - 1) / waves), 64 * waves); };
    bool ok = fits(slots * a.h, 256) && sliced(vtiles, 4) && sliced(vtiles, 8);
    if (a.segment * C < a.n_tokens)
        ok = ok && sliced(vtiles + keys, keys) && sliced(vtiles + keys, 2 * keys) && fits((long long)a.n_seqs * a.h * vtiles, 64 * nk);
    return ok && (!train || fits(slots * a.hk, 512));
}

void launch_delta_fwd(OpType t, DeltaOp a, bool train, hipStream_t s) {
    if (!train && delta_by_token(a)) {
        const long long items = (long long)a.n_seqs * a.h * ((a.dv + 31) / 32);
        for_type(t, [&](auto type) {
            typedef decltype(type) T;
            const dim3 grid(unsigned((items + 3) / 4));
            if (a.dk <= 64) delta_token_kernel<T, 8><<<grid, dim3(256), 0, s>>>(a);
            else delta_token_kernel<T, 16><<<grid, dim3(256), 0, s>>>(a);
        });
        return;
    }
    a.segment = segment_of(t, a, train);
    const int vtiles = 2 * ((a.dv + 31) / 32);
    const bool wide = wide_slices(t, a, a.segment);
    for_type(t, [&](auto type) {
        typedef decltype(type) T;
        for_keys(a.dk, [&](auto nk) {
            for_flag(train, [&](auto training) {
                for_flag(whole_rows(t, a), [&](auto whole) {
                    constexpr bool TRAIN = training.value, WHOLE = whole.value;
                    constexpr int NK = nk.value, C = Parts<T>::C;
                    delta_chunk_kernel<T, NK, WHOLE>
                        <<<dim3(item_grid(slots_on_host(a, C), a.h, 1)), dim3(256), 0, s>>>(a);
                    if (a.segment * C < a.n_tokens) {
                        for_flag(wide && WHOLE, [&](auto both) {
                            constexpr int W = both.value && WHOLE ? 4 * NK : 2 * NK;
                            delta_transit_kernel<T, NK, W, TRAIN, WHOLE>
                                <<<dim3(scan_grid<T>(a, (vtiles + 2 * NK + W - 1) / W)), dim3(64 * W), 0, s>>>(a);
                        });
                        delta_join_kernel<T, NK, false><<<dim3(item_grid(a.n_seqs, a.h, vtiles)), dim3(64 * NK), 0, s>>>(a, a.state_in);
                    }
                    if (wide) delta_scan_kernel<T, NK, 8, TRAIN, WHOLE><<<dim3(scan_grid<T>(a, (vtiles + 7) / 8)), dim3(512), 0, s>>>(a);
                    else delta_scan_kernel<T, NK, 4, TRAIN, WHOLE><<<dim3(scan_grid<T>(a, (vtiles + 3) / 4)), dim3(256), 0, s>>>(a);
                });
            });
        });
    });
}

void launch_delta_bwd(OpType t, DeltaOp a, const DeltaGrad& d, hipStream_t s) {
    a.segment = segment_of(t, a, true);
    const int vtiles = 2 * ((a.dv + 31) / 32);
    const bool aligned = whole_rows(t, a) && reinterpret_cast<uintptr_t>(d.d_o) % 16 == 0, wide = wide_slices(t, a, a.segment);
    for_type(t, [&](auto type) {
        typedef decltype(type) T;
        for_keys(a.dk, [&](auto nk) {
            for_flag(aligned, [&](auto whole) {
                constexpr bool WHOLE = whole.value;
                constexpr int NK = nk.value, C = Parts<T>::C;
                // eight waves as in the scan, where their inputs fit into LDS (two-byte types with aligned rows of more than
                // 64 keys do not)
                constexpr bool FITS = !(WHOLE && NK == 4 && sizeof(T) == 2);
                for_flag(wide && FITS, [&](auto eight) {
                    constexpr int W = eight.value && FITS ? 8 : 4;
                    const dim3 grid(scan_grid<T>(a, (vtiles + W - 1) / W));
                    if (a.segment * C < a.n_tokens) {
                        delta_back_kernel<T, NK, W, true, WHOLE><<<grid, dim3(64 * W), 0, s>>>(a, d);
                        delta_join_kernel<T, NK, true><<<dim3(item_grid(a.n_seqs, a.h, vtiles)), dim3(64 * NK), 0, s>>>(a, d.d_state_out);
                    }
                    delta_back_kernel<T, NK, W, false, WHOLE><<<grid, dim3(64 * W), 0, s>>>(a, d);
                });
                delta_grad_kernel<T, NK, WHOLE><<<dim3(item_grid(slots_on_host(a, C), a.hk, 1)), dim3(512), 0, s>>>(a, d);
            });
        });
    });
}

}  // namespace shv
