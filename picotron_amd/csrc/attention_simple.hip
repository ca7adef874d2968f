// The formulas of attention.h, one wavefront per query row (forward, dq) or key row (dk, dv), fp32 arithmetic.
// A lane computes the scores of one key (row) of a block of 64; for the sums over keys (rows) it owns head columns
// lane, lane + 64, ...  Every product is selected by the mask before it is added, so what is hidden reaches nothing.
#include "attention.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64, kMaxD = 256, kCols = kMaxD / 64;

template <typename T>
__device__ __forceinline__ const T* row_ptr(const AttnTensor& t, int64_t b, int64_t s, int h) {
    return (const T*)t.p + b * t.sb + s * t.ss + h * t.sh;
}

template <typename T>
__device__ __forceinline__ float dot_row(const float* x, const T* y, int D) {
    float sum = 0.f;
    for (int d = 0; d < D; ++d) sum = __builtin_fmaf(x[d], to_f32(y[d]), sum);
    return sum;
}

struct Score {
    float z, slope_of_cap;  // z; dy/dx
};
__device__ __forceinline__ Score score(const AttnArgs& a, float dot, float slope, int pos, int j) {
    float y = dot * a.scale, d = 1.f;
    if (a.softcap > 0.f) {
        const float t = tanhf(y / a.softcap);
        y = a.softcap * t;
        d = 1.f - t * t;
    }
    const int away = pos > j ? pos - j : j - pos;
    return {slope != 0.f ? y - slope * (float)away : y, d};
}

// lse of a row without a key, -inf, as +inf: its P are zeros
__device__ __forceinline__ float no_key_is_infinite(float lse) { return lse == -INFINITY ? INFINITY : lse; }

// the query row a wave works on: its vectors in LDS as floats
struct Row {
    int64_t b;
    int s, h, pos;
    RowSpan span;
    float slope;
    bool in;
};
__device__ __forceinline__ Row wave_row(const AttnArgs& a, int64_t row) {
    Row r;
    r.in = row < a.batch * a.q_len * a.heads;
    if (!r.in) row = 0;
    r.h = (int)(row % a.heads);
    r.s = (int)(row / a.heads % a.q_len);
    r.b = row / a.heads / a.q_len;
    r.pos = r.s + a.kv_len - a.q_len;
    r.span = row_span(a, r.b, r.s);
    r.slope = a.slopes ? a.slopes[r.h] : 0.f;
    return r;
}

__device__ __forceinline__ bool sees(const AttnArgs& a, const RowSpan& r, int64_t b, int j) {
    return j >= r.lo && j <= r.hi && (!a.docs || a.docs[b * a.kv_len + j] == r.doc);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void attention_simple_fwd_kernel(AttnArgs a) {
    __shared__ float qs[kWaves][kMaxD];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * kWaves + wave;
    const Row r = wave_row(a, row);
    const T* q = row_ptr<T>(a.q, r.b, r.s, r.h);
    for (int d = lane; d < a.D; d += 64) qs[wave][d] = to_f32(q[d]);
    __syncthreads();
    if (!r.in) return;
    const int kvh = r.h / a.group;
    float top = -INFINITY, total = 0.f, o[kCols] = {};
    for (int j0 = r.span.lo & ~63; j0 <= r.span.hi; j0 += 64) {
        const int j = j0 + lane;
        const bool ok = sees(a, r.span, r.b, j < a.kv_len ? j : 0) && j < a.kv_len;
        float z = -INFINITY;
        if (ok) z = score(a, dot_row(qs[wave], row_ptr<T>(a.k, r.b, j, kvh), a.D), r.slope, r.pos, j).z;
        const float block_top = wave_max(z), new_top = block_top > top ? block_top : top;
        const float base = new_top == -INFINITY ? 0.f : new_top, shrink = expf(top - base), p = ok ? expf(z - base) : 0.f;
        top = new_top;
        total = total * shrink + wave_sum(p);
        for (int c = 0; c < kCols; ++c) o[c] *= shrink;
        const uint64_t seen = __ballot(ok);
        for (int i = 0; i < 64; ++i) {
            if (!(seen >> i & 1)) continue;
            const float pi = __shfl(p, i, 64);
            const T* v = row_ptr<T>(a.v, r.b, j0 + i, kvh);
            for (int c = 0; c < kCols; ++c)
                if (c * 64 + lane < a.D) o[c] += pi * to_f32(v[c * 64 + lane]);
        }
    }
    // NaN scores leave top at -inf: total is NaN then, and so are the sums
    T* out = (T*)a.out + row * a.D;
    for (int c = 0; c < kCols; ++c)
        if (c * 64 + lane < a.D) {
            const float v = total == 0.f ? 0.f : o[c] / total;
            out[c * 64 + lane] = (T)v;
            if (sizeof(T) == 2 && a.residual) ((T*)a.residual)[row * a.D + c * 64 + lane] = (T)(v - (float)(T)v);
        }
    if (lane == 0) a.lse[(r.b * a.heads + r.h) * a.q_len + r.s] = total == 0.f ? -INFINITY : top + logf(total);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void attention_simple_dq_kernel(AttnArgs a) {
    __shared__ float qs[kWaves][kMaxD], gs[kWaves][kMaxD];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * kWaves + wave;
    const Row r = wave_row(a, row);
    const T* q = row_ptr<T>(a.q, r.b, r.s, r.h);
    const T* g = (const T*)a.d_out + (r.in ? row : 0) * a.D;
    const T* out = (const T*)a.out + (r.in ? row : 0) * a.D;
    float delta = 0.f;
    for (int d = lane; d < a.D; d += 64) {
        qs[wave][d] = to_f32(q[d]);
        gs[wave][d] = to_f32(g[d]);
        float o = to_f32(out[d]);
        if (sizeof(T) == 2 && a.residual) o += to_f32(((const T*)a.residual)[(r.in ? row : 0) * a.D + d]);
        delta += gs[wave][d] * o;
    }
    delta = wave_sum(delta);
    __syncthreads();
    if (!r.in) return;
    const int64_t stat = (r.b * a.heads + r.h) * a.q_len + r.s;
    if (lane == 0) a.delta[stat] = delta;
    const float lse = no_key_is_infinite(a.lse[stat]);
    const int kvh = r.h / a.group;
    float dq[kCols] = {};
    for (int j0 = r.span.lo & ~63; j0 <= r.span.hi; j0 += 64) {
        const int j = j0 + lane;
        const bool ok = sees(a, r.span, r.b, j < a.kv_len ? j : 0) && j < a.kv_len;
        float dx = 0.f;
        if (ok) {
            const Score sc = score(a, dot_row(qs[wave], row_ptr<T>(a.k, r.b, j, kvh), a.D), r.slope, r.pos, j);
            dx = expf(sc.z - lse) * (dot_row(gs[wave], row_ptr<T>(a.v, r.b, j, kvh), a.D) - delta) * sc.slope_of_cap * a.scale;
        }
        const uint64_t seen = __ballot(ok);
        for (int i = 0; i < 64; ++i) {
            if (!(seen >> i & 1)) continue;
            const float di = __shfl(dx, i, 64);
            const T* k = row_ptr<T>(a.k, r.b, j0 + i, kvh);
            for (int c = 0; c < kCols; ++c)
                if (c * 64 + lane < a.D) dq[c] += di * to_f32(k[c * 64 + lane]);
        }
    }
    T* to = (T*)a.dq + row * a.D;
    for (int c = 0; c < kCols; ++c)
        if (c * 64 + lane < a.D) to[c * 64 + lane] = (T)dq[c];
}

template <typename T>
__global__ __launch_bounds__(kThreads) void attention_simple_dkv_kernel(AttnArgs a) {
    __shared__ float ks[kWaves][kMaxD], vs[kWaves][kMaxD];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int64_t key = (int64_t)blockIdx.x * kWaves + wave;
    const bool in = key < a.batch * a.kv_len * a.kv_heads;
    if (!in) key = 0;
    const int kvh = (int)(key % a.kv_heads), j = (int)(key / a.kv_heads % a.kv_len);
    const int64_t b = key / a.kv_heads / a.kv_len;
    const T *k = row_ptr<T>(a.k, b, j, kvh), *v = row_ptr<T>(a.v, b, j, kvh);
    for (int d = lane; d < a.D; d += 64) {
        ks[wave][d] = to_f32(k[d]);
        vs[wave][d] = to_f32(v[d]);
    }
    __syncthreads();
    if (!in) return;
    float dk[kCols] = {}, dv[kCols] = {};
    const int64_t rows = (int64_t)a.q_len * a.group;
    for (int64_t r0 = 0; r0 < rows; r0 += 64) {
        const int64_t row = r0 + lane;
        const int s = (int)(row / a.group), h = kvh * a.group + (int)(row % a.group);
        bool ok = row < rows;
        const RowSpan span = row_span(a, b, ok ? s : 0);
        ok = ok && sees(a, span, b, j);
        float p = 0.f, dx = 0.f;
        if (ok) {
            const int64_t stat = (b * a.heads + h) * a.q_len + s;
            const Score sc = score(a, dot_row(ks[wave], row_ptr<T>(a.q, b, s, h), a.D), a.slopes ? a.slopes[h] : 0.f, s + a.kv_len - a.q_len, j);
            p = expf(sc.z - no_key_is_infinite(a.lse[stat]));
            const T* g = (const T*)a.d_out + ((b * a.q_len + s) * a.heads + h) * a.D;
            dx = p * (dot_row(vs[wave], g, a.D) - a.delta[stat]) * sc.slope_of_cap * a.scale;
        }
        const uint64_t seen = __ballot(ok);
        for (int i = 0; i < 64; ++i) {
            if (!(seen >> i & 1)) continue;
            const float pi = __shfl(p, i, 64), di = __shfl(dx, i, 64);
            const int si = (int)((r0 + i) / a.group), hi = kvh * a.group + (int)((r0 + i) % a.group);
            const T* q = row_ptr<T>(a.q, b, si, hi);
            const T* g = (const T*)a.d_out + ((b * a.q_len + si) * a.heads + hi) * a.D;
            for (int c = 0; c < kCols; ++c) {
                if (c * 64 + lane >= a.D) continue;
                dk[c] += di * to_f32(q[c * 64 + lane]);
                dv[c] += pi * to_f32(g[c * 64 + lane]);
            }
        }
    }
    for (int c = 0; c < kCols; ++c) {
        if (c * 64 + lane >= a.D) continue;
        ((T*)a.dk)[key * a.D + c * 64 + lane] = (T)dk[c];
        ((T*)a.dv)[key * a.D + c * 64 + lane] = (T)dv[c];
    }
}

}  // namespace

int attention_simple_fwd(const AttnArgs& a, hipStream_t s) {
    const int64_t blocks = (a.batch * a.q_len * a.heads + kWaves - 1) / kWaves;
    if (blocks > 0x7FFFFFFF) return PICOMOE_ERR_TOO_LARGE;
    if (a.dtype == PICOMOE_BF16) attention_simple_fwd_kernel<__bf16><<<(unsigned)blocks, kThreads, 0, s>>>(a);
    else attention_simple_fwd_kernel<float><<<(unsigned)blocks, kThreads, 0, s>>>(a);
    return picomoe_launch_status();
}

int attention_simple_bwd(const AttnArgs& a, hipStream_t s) {
    const int64_t blocks = (a.batch * a.q_len * a.heads + kWaves - 1) / kWaves, key_blocks = (a.batch * a.kv_len * a.kv_heads + kWaves - 1) / kWaves;
    if (blocks > 0x7FFFFFFF || key_blocks > 0x7FFFFFFF) return PICOMOE_ERR_TOO_LARGE;
    if (a.dtype == PICOMOE_BF16) {
        attention_simple_dq_kernel<__bf16><<<(unsigned)blocks, kThreads, 0, s>>>(a);
        attention_simple_dkv_kernel<__bf16><<<(unsigned)key_blocks, kThreads, 0, s>>>(a);
    } else {
        attention_simple_dq_kernel<float><<<(unsigned)blocks, kThreads, 0, s>>>(a);
        attention_simple_dkv_kernel<float><<<(unsigned)key_blocks, kThreads, 0, s>>>(a);
    }
    return picomoe_launch_status();
}
