// extern "C" entry points of the attention: checks of the arguments, the layout of the workspaces, the choice of kernels.
#include "attention.h"

namespace {

constexpr int64_t kMaxLength = 1 << 28;

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

bool sizes_ok(int dtype, int64_t batch, int64_t q_len, int64_t kv_len, int q_heads, int kv_heads, int head_dim) {
    return (dtype == PICOMOE_F32 || dtype == PICOMOE_BF16) && batch >= 0 && batch <= 1 << 24 && q_len >= 0 && q_len <= kMaxLength && kv_len >= 0 &&
           kv_len <= kMaxLength && q_heads >= 1 && q_heads <= 4096 && kv_heads >= 1 && q_heads % kv_heads == 0 && head_dim >= 8 && head_dim <= 256 &&
           head_dim % 8 == 0 && q_len * (q_heads / kv_heads) <= (1ll << 30);
}

bool tensor(AttnTensor* t, const void* p, const int64_t* strides, int dtype) {
    const int64_t vec = dtype == PICOMOE_BF16 ? 8 : 4;  // elements of a 16-byte access
    if (!p || !strides || ((uintptr_t)p & 15) || strides[0] % vec || strides[1] % vec || strides[2] % vec) return false;
    if (strides[0] < 0 || strides[1] < 0 || strides[2] < 0) return false;  // offsets inside a tile are unsigned
    *t = {p, strides[0], strides[1], strides[2]};
    return true;
}

bool fill(AttnArgs* a, const void* q, const int64_t* qs, const void* k, const int64_t* ks, const void* v, const int64_t* vs, int dtype, int64_t batch,
          int64_t q_len, int64_t kv_len, int q_heads, int kv_heads, int head_dim, float scale, float softcap, int causal, int64_t window,
          const float* slopes, const int32_t* docs, const int32_t* prefix) {
    if (!(softcap >= 0.f) || softcap > 1e30f || !(scale >= -3e38f && scale <= 3e38f) || window < 0 || (prefix && !causal)) return false;
    if (softcap > 0.f && scale != 0.f) {  // the factor of q . k inside the cap: normal, and finite times 2 log2(e)
        const float inside = (scale < 0.f ? -scale : scale) / softcap;
        if (!(inside >= 1.2e-38f && inside < 1e38f)) return false;
    }
    if (!tensor(&a->q, q, qs, dtype)) return false;
    if (kv_len > 0 && (!tensor(&a->k, k, ks, dtype) || !tensor(&a->v, v, vs, dtype))) return false;
    a->dtype = dtype; a->causal = causal != 0; a->batch = batch;
    a->q_len = (int)q_len; a->kv_len = (int)kv_len; a->heads = q_heads; a->kv_heads = kv_heads; a->group = q_heads / kv_heads; a->D = head_dim;
    a->scale = scale; a->softcap = softcap;
    a->window = window >= q_len + kv_len ? 0 : (int)window;  // no query is that far from a key
    a->slopes = slopes; a->docs = docs; a->prefix = prefix;
    return true;
}

}  // namespace

extern "C" int64_t picomoe_attention_fwd_workspace_bytes(int dtype, int64_t batch, int64_t q_len, int64_t kv_len, int q_heads, int kv_heads,
                                                         int head_dim) {
    if (!sizes_ok(dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim)) return -1;
    return attention_mfma_supported(dtype, head_dim) ? attention_mfma_fwd_workspace(dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim) : 16;
}

extern "C" int picomoe_attention_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                                     const int64_t* v_strides, int dtype, int64_t batch, int64_t q_len, int64_t kv_len, int q_heads, int kv_heads,
                                     int head_dim, float scale, float softcap, int causal, int64_t window, const float* slopes,
                                     const int32_t* document_ids, const int32_t* prefix_lengths, void* out, void* out_residual, float* lse, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
    PICOMOE_CHECK_ARG(sizes_ok(dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim));
    if (batch == 0 || q_len == 0) return PICOMOE_OK;
    AttnArgs a = {};
    PICOMOE_CHECK_ARG(fill(&a, q, q_strides, k, k_strides, v, v_strides, dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim, scale, softcap,
                           causal, window, slopes, document_ids, prefix_lengths));
    PICOMOE_CHECK_ARG(out && lse && (((uintptr_t)out | (uintptr_t)out_residual) & 15) == 0 && workspace && ((uintptr_t)workspace & 15) == 0 &&
                      workspace_bytes >= picomoe_attention_fwd_workspace_bytes(dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim));
    a.out = out; a.residual = dtype == PICOMOE_BF16 ? out_residual : nullptr; a.lse = lse; a.ws = (char*)workspace;
    if (attention_mfma_supported(dtype, head_dim)) return attention_mfma_fwd(a, (hipStream_t)stream);
    return attention_simple_fwd(a, (hipStream_t)stream);
}

extern "C" int64_t picomoe_attention_bwd_workspace_bytes(int dtype, int64_t batch, int64_t q_len, int64_t kv_len, int q_heads, int kv_heads,
                                                         int head_dim) {
    if (!sizes_ok(dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim)) return -1;
    if (attention_mfma_supported(dtype, head_dim)) return attention_mfma_bwd_workspace(dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim);
    return round16(batch * q_len * q_heads * 4) + 16;  // D of the rows
}

extern "C" int picomoe_attention_bwd(const void* d_out, const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                                     const int64_t* v_strides, const void* out, const void* out_residual, const float* lse, int dtype, int64_t batch, int64_t q_len,
                                     int64_t kv_len, int q_heads, int kv_heads, int head_dim, float scale, float softcap, int causal, int64_t window,
                                     const float* slopes, const int32_t* document_ids, const int32_t* prefix_lengths, void* dq, void* dk, void* dv,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
    PICOMOE_CHECK_ARG(sizes_ok(dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim) && q_len > 0 && kv_len > 0);
    if (batch == 0) return PICOMOE_OK;
    AttnArgs a = {};
    PICOMOE_CHECK_ARG(fill(&a, q, q_strides, k, k_strides, v, v_strides, dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim, scale, softcap,
                           causal, window, slopes, document_ids, prefix_lengths));
    auto ok16 = [](const void* p) { return p && ((uintptr_t)p & 15) == 0; };
    PICOMOE_CHECK_ARG(ok16(d_out) && ok16(out) && ((uintptr_t)out_residual & 15) == 0 && lse && ok16(dq) && ok16(dk) && ok16(dv) && ok16(workspace) &&
                      workspace_bytes >= picomoe_attention_bwd_workspace_bytes(dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim));
    a.out = (void*)out; a.residual = dtype == PICOMOE_BF16 ? (void*)out_residual : nullptr; a.lse = (float*)lse; a.d_out = d_out; a.dq = dq; a.dk = dk; a.dv = dv;
    a.delta = (float*)workspace;
    a.ws = (char*)workspace;
    if (attention_mfma_supported(dtype, head_dim)) return attention_mfma_bwd(a, (hipStream_t)stream);
    return attention_simple_bwd(a, (hipStream_t)stream);
}
