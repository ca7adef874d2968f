// RMS norm of each query and key head and the position rotation, in one pass over the heads, and its gradient.
//
// Per head row x of D values (D even, halves a = x[:D/2], b = x[D/2:]), with weight w and table rows c, s at its position:
//
//   r = rsqrt(mean(x^2) + eps)      n = r x      y = w n          (no weight: y = x)
//   out[i] = y[i] c[i] - y[i + D/2] s[i]          out[i + D/2] = y[i + D/2] c[i + D/2] + y[i] s[i + D/2]
//
// Backward, g = d out:
//   dy[i] = g[i] c[i] + g[i + D/2] s[i + D/2]     dy[i + D/2] = g[i + D/2] c[i + D/2] - g[i] s[i]
//   dn = w dy      dx = r (dn - n mean(dn n))      dw = sum over rows of dy n
//
// Everything is computed in fp32 and rounded once, at the store.  Both passes are bound by memory: forward one read and one
// write of the heads, backward two reads (x and g; r is recomputed, nothing is saved) and one write.  A lane holds kVec values
// of the first half and the kVec values they are rotated with, so the rotation needs no exchange and the sum of squares one
// butterfly over the lanes of a head.  A group of lanes takes some heads of one token, whose table rows it reads once -- in fp32
// they are twice a bf16 head --, and has the loads of all of them in flight.  Queries and keys go through one launch.  dw is summed
// in registers over the rows a group walks, joined per block in LDS and over the blocks by a second launch, in a fixed order.
// Measured, bf16, 8192 tokens x (32 + 8) heads of 128: forward 36 us (168 MB: 4.7 TB/s), backward 58 us (252 MB: 4.3 TB/s) + 5 us for
// dw; a large copy runs at 4.9 TB/s.  One token of 16 sequences: 6 us, a launch.
#include "common.h"

namespace {

constexpr int kThreads = 256;

template <typename T, int VEC>
struct Vec;
template <>
struct Vec<__bf16, 8> {
    typedef u32x4_t raw;
    __device__ static void get(const raw& r, float (&f)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    __device__ static raw put(const float (&f)[8]) {
        return raw{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
    }
};
template <>
struct Vec<__bf16, 4> {
    typedef u32x2_t raw;
    __device__ static void get(const raw& r, float (&f)[4]) {
        f[0] = __uint_as_float(r.x << 16);
        f[1] = __uint_as_float(r.x & 0xFFFF0000u);
        f[2] = __uint_as_float(r.y << 16);
        f[3] = __uint_as_float(r.y & 0xFFFF0000u);
    }
    __device__ static raw put(const float (&f)[4]) { return raw{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3])}; }
};
template <>
struct Vec<float, 4> {
    typedef f32x4_t raw;
    __device__ static void get(const raw& r, float (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = r[i];
    }
    __device__ static raw put(const float (&f)[4]) { return raw{f[0], f[1], f[2], f[3]}; }
};

struct Heads {  // queries or keys: [batch, seq, heads, D] with strides in elements, last dimension dense
    const void* x;
    const void* grad;     // backward: [batch, seq, heads, D], dense
    const void* weight;   // NULL: no norm
    void* out;            // dense
    int64_t sb, ss, sh;
    int heads;
};

struct Args {
    Heads q, k;
    const float *cos, *sin;     // [n_positions, D]
    const int64_t* positions;   // [batch, seq] or NULL: the token's place in its row
    int64_t n_positions, tokens, seq;
    float eps;
    int D;
    float* partial;  // backward: [blocks][2][D] sums of dw
};

// field by field: a reference to one of the two would put the arguments into scratch memory
__device__ __forceinline__ Heads pick(const Args& a, bool k) {
    return {k ? a.k.x : a.q.x, k ? a.k.grad : a.q.grad, k ? a.k.weight : a.q.weight, k ? a.k.out : a.q.out, k ? a.k.sb : a.q.sb,
            k ? a.k.ss : a.q.ss, k ? a.k.sh : a.q.sh, k ? a.k.heads : a.q.heads};
}

// A group of `lanes` lanes holds a head.
template <typename T, int VEC>
struct Lane {
    typedef Vec<T, VEC> V;
    typedef typename V::raw raw;
    int half, col;   // this lane's first column, below half
    bool in;         // lanes past half / VEC of a group read the first lane's and hold zeros

    __device__ Lane(int D, int lanes) {
        half = D / 2;
        const int l = threadIdx.x & (lanes - 1);
        in = l * VEC < half;
        col = in ? l * VEC : 0;
    }
    __device__ void load(const T* p, float (&a)[VEC], float (&b)[VEC]) const {
        V::get(*(const raw*)(p + col), a);
        V::get(*(const raw*)(p + half + col), b);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            a[i] = in ? a[i] : 0.f;
            b[i] = in ? b[i] : 0.f;
        }
    }
    __device__ void store(T* p, const float (&a)[VEC], const float (&b)[VEC]) const {
        if (in) {
            *(raw*)(p + col) = V::put(a);
            *(raw*)(p + half + col) = V::put(b);
        }
    }
    __device__ void load_f32(const float* p, float (&a)[VEC], float (&b)[VEC]) const {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const f32x4_t u = *(const f32x4_t*)(p + col + i), v = *(const f32x4_t*)(p + half + col + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a[i + j] = u[j];
                b[i + j] = v[j];
            }
        }
    }
};

__device__ __forceinline__ float group_sum(float v, int lanes) {
    for (int off = lanes >> 1; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// The table rows of a token; NaN where its position has none, so that a bad position shows in its outputs and gradients
template <typename T, int VEC>
__device__ __forceinline__ void table_rows(const Args& a, const Lane<T, VEC>& ln, int64_t token, float (&c0)[VEC], float (&c1)[VEC],
                                           float (&s0)[VEC], float (&s1)[VEC]) {
    const int64_t pos = a.positions ? a.positions[token] : token % a.seq;
    const bool good = pos >= 0 && pos < a.n_positions;
    const int64_t at = good ? pos * a.D : 0;
    ln.load_f32(a.cos + at, c0, c1);
    ln.load_f32(a.sin + at, s0, s1);
    const float nan = __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        c0[i] = good ? c0[i] : nan;
        c1[i] = good ? c1[i] : nan;
        s0[i] = good ? s0[i] : nan;
        s1[i] = good ? s1[i] : nan;
    }
}

template <typename T, int VEC>
__device__ __forceinline__ float row_rms(const float (&a)[VEC], const float (&b)[VEC], int lanes, int D, float eps) {
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) sq += a[i] * a[i] + b[i] * b[i];
    return 1.0f / sqrtf(group_sum(sq, lanes) / (float)D + eps);
}

// Heads that a group has in flight.  The backward, which loads two rows a head, takes 59 us with one at 8192 tokens x (32 + 8) heads of
// 128, 78 with two and 80 with four: the registers cost it more waves than the loads in flight bring.
constexpr int kFwdHeads = 4, kBwdHeads = 1;

// Work is numbered token by token, and in a token by sets of kFwdHeads query heads, then of key heads.
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_fwd_kernel(Args a, int lanes) {
    const Lane<T, VEC> ln(a.D, lanes);
    const int q_sets = (a.q.heads + kFwdHeads - 1) / kFwdHeads, sets = q_sets + (a.k.heads + kFwdHeads - 1) / kFwdHeads;
    const int64_t set = (int64_t)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes, token = set / sets;
    if (token >= a.tokens) return;
    const int in_token = (int)(set - token * sets);
    const bool is_k = in_token >= q_sets;
    const Heads t = pick(a, is_k);
    const int h0 = (is_k ? in_token - q_sets : in_token) * kFwdHeads, n = min(kFwdHeads, t.heads - h0);
    const int64_t b = token / a.seq, s = token - b * a.seq;
    const T* x = (const T*)t.x + b * t.sb + s * t.ss + h0 * t.sh;
    float x0[kFwdHeads][VEC], x1[kFwdHeads][VEC], c0[VEC], c1[VEC], s0[VEC], s1[VEC], w0[VEC], w1[VEC];
#pragma unroll
    for (int h = 0; h < kFwdHeads; ++h)
        if (h < n) ln.load(x + h * t.sh, x0[h], x1[h]);
    table_rows<T, VEC>(a, ln, token, c0, c1, s0, s1);
    if (t.weight) ln.load((const T*)t.weight, w0, w1);
#pragma unroll
    for (int h = 0; h < kFwdHeads; ++h) {
        if (h >= n) break;
        if (t.weight) {
            const float r = row_rms<T, VEC>(x0[h], x1[h], lanes, a.D, a.eps);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                x0[h][i] = x0[h][i] * r * w0[i];
                x1[h][i] = x1[h][i] * r * w1[i];
            }
        }
        float o0[VEC], o1[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            o0[i] = x0[h][i] * c0[i] - x1[h][i] * s0[i];
            o1[i] = x1[h][i] * c1[i] + x0[h][i] * s1[i];
        }
        ln.store((T*)t.out + (token * t.heads + h0 + h) * a.D, o0, o1);
    }
}

// A group walks sets of one tensor only -- the first q_blocks blocks the queries, the others the keys -- and keeps its columns of dw.
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_bwd_kernel(Args a, int lanes, int q_blocks) {
    const Lane<T, VEC> ln(a.D, lanes);
    const bool is_k = (int)blockIdx.x >= q_blocks;
    const Heads t = pick(a, is_k);
    const int groups = kThreads / lanes, group = threadIdx.x / lanes, sets = (t.heads + kBwdHeads - 1) / kBwdHeads;
    const int64_t block = is_k ? blockIdx.x - q_blocks : blockIdx.x, blocks = is_k ? gridDim.x - q_blocks : q_blocks;
    float w0[VEC], w1[VEC], dw0[VEC], dw1[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw0[i] = dw1[i] = 0.f;
    if (t.weight) ln.load((const T*)t.weight, w0, w1);
    for (int64_t set = block * groups + group; set < a.tokens * sets; set += blocks * groups) {
        const int64_t token = set / sets, b = token / a.seq, s = token - b * a.seq;
        const int h0 = (int)(set - token * sets) * kBwdHeads, n = min(kBwdHeads, t.heads - h0);
        const int64_t row = token * t.heads + h0;
        const T* x = (const T*)t.x + b * t.sb + s * t.ss + h0 * t.sh;
        float x0[kBwdHeads][VEC], x1[kBwdHeads][VEC], g0[kBwdHeads][VEC], g1[kBwdHeads][VEC], c0[VEC], c1[VEC], s0[VEC], s1[VEC];
#pragma unroll
        for (int h = 0; h < kBwdHeads; ++h) {
            if (h >= n) break;
            ln.load((const T*)t.grad + (row + h) * a.D, g0[h], g1[h]);
            if (t.weight) ln.load(x + h * t.sh, x0[h], x1[h]);
        }
        table_rows<T, VEC>(a, ln, token, c0, c1, s0, s1);
#pragma unroll
        for (int h = 0; h < kBwdHeads; ++h) {
            if (h >= n) break;
            float y0[VEC], y1[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                y0[i] = g0[h][i] * c0[i] + g1[h][i] * s1[i];
                y1[i] = g1[h][i] * c1[i] - g0[h][i] * s0[i];
            }
            if (t.weight) {
                const float r = row_rms<T, VEC>(x0[h], x1[h], lanes, a.D, a.eps);
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    x0[h][i] *= r;
                    x1[h][i] *= r;
                    dw0[i] += y0[i] * x0[h][i];
                    dw1[i] += y1[i] * x1[h][i];
                    y0[i] *= w0[i];
                    y1[i] *= w1[i];
                    dot += y0[i] * x0[h][i] + y1[i] * x1[h][i];
                }
                dot = group_sum(ln.in ? dot : 0.f, lanes) / (float)a.D;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    y0[i] = r * (y0[i] - x0[h][i] * dot);
                    y1[i] = r * (y1[i] - x1[h][i] * dot);
                }
            }
            ln.store((T*)t.out + (row + h) * a.D, y0, y1);
        }
    }
    if (!a.partial || !t.weight) return;
    extern __shared__ float sums[];  // [groups][D]
    if (ln.in) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            sums[group * a.D + ln.col + i] = dw0[i];
            sums[group * a.D + ln.half + ln.col + i] = dw1[i];
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.D; c += kThreads) {
        float sum = 0.f;
        for (int g = 0; g < groups; ++g) sum += sums[g * a.D + c];
        a.partial[(int64_t)blockIdx.x * a.D + c] = sum;
    }
}

// dw: blockIdx.y 0 for the queries, 1 for the keys, 16 columns a block; 64 threads per column sum consecutive blocks' parts
constexpr int kGradColumns = 16;
template <typename T>
__global__ __launch_bounds__(1024) void qk_weight_grad_kernel(const float* __restrict__ partial, int D, int q_blocks, int k_blocks, T* dq_weight,
                                                              T* dk_weight) {
    __shared__ float part[64][kGradColumns + 1];
    T* out = blockIdx.y ? dk_weight : dq_weight;
    if (!out) return;
    const int first = blockIdx.y ? q_blocks : 0, count = blockIdx.y ? k_blocks : q_blocks;
    const int c = threadIdx.x % kGradColumns, col = blockIdx.x * kGradColumns + c, slice = threadIdx.x / kGradColumns, per = (count + 63) / 64;
    const int from = slice * per, to = min(from + per, count);
    float sum = 0.f;
    if (col < D) {
#pragma unroll 8
        for (int b = from; b < to; ++b) sum += partial[(int64_t)(first + b) * D + col];
    }
    part[slice][c] = sum;
    __syncthreads();
    if (slice != 0 || col >= D) return;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) sum += part[i][c];
    out[col] = (T)sum;
}

// ---------------------------------------------------------------------------------------------------------------
constexpr int kMaxBlocks = 2048;  // of the backward, queries and keys together

int lanes_for(int D, int vec) {
    int lanes = 1;
    while (lanes * vec < D / 2) lanes *= 2;
    return lanes;
}

bool aligned(const void* p, int64_t bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

bool valid(int dtype, int64_t batch, int64_t seq, int q_heads, int k_heads, int head_dim) {
    return (dtype == PICOMOE_F32 || dtype == PICOMOE_BF16) && batch >= 0 && seq >= 0 && q_heads >= 1 && k_heads >= 1 && q_heads <= 4096 &&
           k_heads <= 4096 && head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0 && (seq == 0 || batch < (1ll << 31) / seq);
}

// 16-byte accesses need D / 2 to be a whole number of them and every row to start on one; 8-byte ones are left for bf16 otherwise
int vec_for(int dtype, int D, const Heads& q, const Heads& k) {
    if (dtype == PICOMOE_F32) return 4;
    auto fits = [](const Heads& t) { return aligned(t.x, 16) && t.sb % 8 == 0 && t.ss % 8 == 0 && t.sh % 8 == 0 && aligned(t.weight, 16); };
    return D % 16 == 0 && fits(q) && fits(k) ? 8 : 4;
}

bool heads_ok(const Heads& t, int dtype, bool backward) {
    const int64_t bytes = dtype == PICOMOE_F32 ? 16 : 8;
    return t.x && t.out && t.sb % 4 == 0 && t.ss % 4 == 0 && t.sh % 4 == 0 && aligned(t.x, bytes) && aligned(t.out, 16) && aligned(t.weight, bytes) &&
           (!backward || (t.grad && aligned(t.grad, 16)));
}

struct Blocks {
    int q, k;
};
int64_t head_sets(int heads, int per) { return (heads + per - 1) / per; }
Blocks bwd_blocks(int64_t tokens, int q_heads, int k_heads, int lanes) {
    const int64_t groups = kThreads / lanes, q_sets = head_sets(q_heads, kBwdHeads), k_sets = head_sets(k_heads, kBwdHeads);
    const int64_t q_need = (tokens * q_sets + groups - 1) / groups, k_need = (tokens * k_sets + groups - 1) / groups;
    if (q_need + k_need <= kMaxBlocks) return {(int)q_need, (int)k_need};
    int q = (int)(kMaxBlocks * q_sets / (q_sets + k_sets));
    q = q < 1 ? 1 : (q > kMaxBlocks - 1 ? kMaxBlocks - 1 : q);
    return {q, kMaxBlocks - q};
}

template <typename T, int VEC>
int launch_fwd(const Args& a, hipStream_t s) {
    const int lanes = lanes_for(a.D, VEC), groups = kThreads / lanes;
    const int64_t blocks = (a.tokens * (head_sets(a.q.heads, kFwdHeads) + head_sets(a.k.heads, kFwdHeads)) + groups - 1) / groups;
    if (blocks > 0x7FFFFFFF) return PICOMOE_ERR_TOO_LARGE;
    qk_norm_rope_fwd_kernel<T, VEC><<<(unsigned)blocks, kThreads, 0, s>>>(a, lanes);
    return picomoe_launch_status();
}

template <typename T, int VEC>
int launch_bwd(const Args& a, void* dq_weight, void* dk_weight, hipStream_t s) {
    const int lanes = lanes_for(a.D, VEC);
    const Blocks n = bwd_blocks(a.tokens, a.q.heads, a.k.heads, lanes);
    if (n.q + n.k > 0)
        qk_norm_rope_bwd_kernel<T, VEC><<<(unsigned)(n.q + n.k), kThreads, kThreads / lanes * a.D * sizeof(float), s>>>(a, lanes, n.q);
    if (dq_weight || dk_weight) qk_weight_grad_kernel<T><<<dim3((unsigned)((a.D + kGradColumns - 1) / kGradColumns), 2), 1024, 0, s>>>(a.partial, a.D, n.q, n.k, (T*)dq_weight, (T*)dk_weight);
    return picomoe_launch_status();
}

}  // namespace

extern "C" int picomoe_qk_norm_rope_fwd(const void* q, const int64_t* q_strides, int q_heads, const void* k, const int64_t* k_strides, int k_heads,
                                        int dtype, int64_t batch, int64_t seq, int head_dim, const void* q_weight, const void* k_weight, float eps,
                                        const float* cos, const float* sin, int64_t n_positions, const int64_t* positions, void* q_out, void* k_out,
                                        void* stream) {
    PICOMOE_CHECK_ARG(valid(dtype, batch, seq, q_heads, k_heads, head_dim) && q_strides && k_strides && n_positions >= 0 && eps >= 0.f && eps <= 3e38f);
    if (batch == 0 || seq == 0) return PICOMOE_OK;
    Args a = {};
    a.q = {q, nullptr, q_weight, q_out, q_strides[0], q_strides[1], q_strides[2], q_heads};
    a.k = {k, nullptr, k_weight, k_out, k_strides[0], k_strides[1], k_strides[2], k_heads};
    PICOMOE_CHECK_ARG(heads_ok(a.q, dtype, false) && heads_ok(a.k, dtype, false) && cos && sin && n_positions > 0 && aligned(cos, 16) && aligned(sin, 16));
    a.cos = cos; a.sin = sin; a.positions = positions; a.n_positions = n_positions;
    a.tokens = batch * seq; a.seq = seq; a.eps = eps; a.D = head_dim;
    if (dtype == PICOMOE_F32) return launch_fwd<float, 4>(a, (hipStream_t)stream);
    return vec_for(dtype, head_dim, a.q, a.k) == 8 ? launch_fwd<__bf16, 8>(a, (hipStream_t)stream) : launch_fwd<__bf16, 4>(a, (hipStream_t)stream);
}

extern "C" int64_t picomoe_qk_norm_rope_bwd_workspace_bytes(int dtype, int64_t batch, int64_t seq, int q_heads, int k_heads, int head_dim) {
    if (!valid(dtype, batch, seq, q_heads, k_heads, head_dim)) return -1;
    const Blocks n = bwd_blocks(batch * seq, q_heads, k_heads, lanes_for(head_dim, 4));  // the narrower accesses have the more blocks
    return ((int64_t)(n.q + n.k) * head_dim * 4 + 15) / 16 * 16;
}

extern "C" int picomoe_qk_norm_rope_bwd(const void* dq_out, const void* dk_out, const void* q, const int64_t* q_strides, int q_heads, const void* k,
                                        const int64_t* k_strides, int k_heads, int dtype, int64_t batch, int64_t seq, int head_dim,
                                        const void* q_weight, const void* k_weight, float eps, const float* cos, const float* sin,
                                        int64_t n_positions, const int64_t* positions, void* dq, void* dk, void* dq_weight, void* dk_weight,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
    PICOMOE_CHECK_ARG(valid(dtype, batch, seq, q_heads, k_heads, head_dim) && q_strides && k_strides && n_positions >= 0 && eps >= 0.f && eps <= 3e38f);
    PICOMOE_CHECK_ARG((!dq_weight || q_weight) && (!dk_weight || k_weight));
    Args a = {};
    a.q = {q, dq_out, q_weight, dq, q_strides[0], q_strides[1], q_strides[2], q_heads};
    a.k = {k, dk_out, k_weight, dk, k_strides[0], k_strides[1], k_strides[2], k_heads};
    const bool empty = batch == 0 || seq == 0;
    PICOMOE_CHECK_ARG(empty || (heads_ok(a.q, dtype, true) && heads_ok(a.k, dtype, true) && cos && sin && n_positions > 0 && aligned(cos, 16) && aligned(sin, 16)));
    if (dq_weight || dk_weight) {
        PICOMOE_CHECK_ARG(empty || (workspace && aligned(workspace, 16) &&
                                    workspace_bytes >= picomoe_qk_norm_rope_bwd_workspace_bytes(dtype, batch, seq, q_heads, k_heads, head_dim)));
        a.partial = (float*)workspace;
    }
    a.cos = cos; a.sin = sin; a.positions = positions; a.n_positions = n_positions;
    a.tokens = batch * seq; a.seq = seq > 0 ? seq : 1; a.eps = eps; a.D = head_dim;
    if (dtype == PICOMOE_F32) return launch_bwd<float, 4>(a, dq_weight, dk_weight, (hipStream_t)stream);
    return vec_for(dtype, head_dim, a.q, a.k) == 8 ? launch_bwd<__bf16, 8>(a, dq_weight, dk_weight, (hipStream_t)stream)
                                                   : launch_bwd<__bf16, 4>(a, dq_weight, dk_weight, (hipStream_t)stream);
}
