// Grouped-query attention with capped scores, distance bias and structural masks: what its kernels share.
//
// Query s of head h stands at position p = s + kv_len - q_len.  Over the keys j that it sees,
//
//   x[j] = scale q . k[j]      y[j] = softcap tanh(x[j] / softcap)  (softcap 0: y = x)      z[j] = y[j] - slope[h] |p - j|
//   P[j] = exp(z[j]) / sum exp(z)          out = sum P[j] v[j]          lse = log sum exp(z)
//
// and a query that sees no key -- or has only scores of -inf -- gets out = 0, lse = -inf.  Which keys: an interval [lo, hi] (causal: j <= p, or j < prefix length;
// window: |p - j| < window), and of those the ones of the query's document (equal ids, not negative).  A key outside takes no
// part at all: NaN or infinity in its k or v (or in the q or d_out of a query that does not see the key) reaches nothing.
//
// Backward, g = d out:   D = g . out (with the residual of out, where it is bf16: D's error would reach every dx of the row)
//       dP[j] = g . v[j]      dz = P (dP - D)      dx = dz (1 - (y / softcap)^2)
//   dq = scale sum dx[j] k[j]      dk[j] = scale sum over queries and heads of the group of dx q      dv[j] = sum P[j] g
#pragma once
#include "common.h"

struct AttnTensor {  // [batch, length, heads, head_dim]: strides in elements, last dimension dense
    const void* p;
    int64_t sb, ss, sh;
};

struct AttnArgs {
    AttnTensor q, k, v;
    int dtype, causal;
    int64_t batch;
    int q_len, kv_len, heads, kv_heads, group, D;  // group: query heads per key head
    float scale, softcap;                          // softcap 0: none
    int window;                                    // 0: none
    const float* slopes;                           // [heads] or NULL
    const int32_t* docs;                           // [batch, kv_len] or NULL
    const int32_t* prefix;                         // [batch] or NULL
    void* out;                                     // [batch, q_len, heads, D]
    float* lse;                                    // [batch, heads, q_len], natural log
    void* residual;                                // like out: what its rounding to bf16 left, rounded to bf16; or NULL
    // backward
    const void* d_out;
    void *dq, *dk, *dv;
    float* delta;  // the simple kernels' workspace, [batch, heads, q_len]: D above
    char* ws;      // the MFMA kernels' workspace
};

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct RowSpan {
    int lo, hi;  // keys the query may see, hi < lo: none
    int doc;
};

__device__ __forceinline__ RowSpan row_span(const AttnArgs& a, int64_t b, int s) {
    const int pos = s + (a.kv_len - a.q_len);
    RowSpan r = {0, a.kv_len - 1, 0};
    if (a.causal) {
        int last = pos;
        if (a.prefix) {
            const int pre = (a.prefix[b] > 0 ? a.prefix[b] : 0) - 1;
            last = pre > last ? pre : last;
        }
        r.hi = last < r.hi ? last : r.hi;
    }
    if (a.window > 0) {
        r.lo = pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
        r.hi = pos + a.window - 1 < r.hi ? pos + a.window - 1 : r.hi;
    }
    if (a.docs) {
        r.doc = pos >= 0 ? a.docs[b * a.kv_len + pos] : -1;
        if (r.doc < 0) r.hi = -1, r.lo = 0;
    }
    return r;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__bf16>(__bf16 v) { return (float)v; }

}  // namespace

int attention_simple_fwd(const AttnArgs& a, hipStream_t s);
int attention_simple_bwd(const AttnArgs& a, hipStream_t s);
// The MFMA kernels (attention_fwd.hip, attention_bwd.hip): head_dim up to 128, in bf16 up to 256.  A tile of fp32 rows of 256 and what
// goes with it are beyond a CU's LDS.
bool attention_mfma_supported(int dtype, int head_dim);
int64_t attention_mfma_fwd_workspace(int dtype, int64_t batch, int64_t q_len, int64_t kv_len, int q_heads, int kv_heads, int head_dim);
int attention_mfma_fwd(const AttnArgs& a, hipStream_t s);
int64_t attention_mfma_bwd_workspace(int dtype, int64_t batch, int64_t q_len, int64_t kv_len, int q_heads, int kv_heads, int head_dim);
int attention_mfma_bwd(const AttnArgs& a, hipStream_t s);
