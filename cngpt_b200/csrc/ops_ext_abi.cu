// ops_ext_abi.cu - C entry points of the operators on a model's distribution
// and of the shared-prefix decode attention (cngpt_cuda.h): the checks of the
// arguments, then the launchers of kernels.h on the library stream. All
// pointers are device (or managed) pointers; nothing is staged.
#include <cmath>

#include "abi_common.h"
#include "kernels.h"

extern "C" {
#include "cngpt_cuda.h"
}

namespace cg {

int dev_ptr(const char *fn, const char *name, const void *p) {
    if (!p) {
        set_last_error(ERR_ARG, "%s: %s is NULL", fn, name);
        return ERR_ARG;
    }
    if ((uintptr_t)p % 4) {
        set_last_error(ERR_ARG, "%s: %s is not 4-byte aligned", fn, name);
        return ERR_ARG;
    }
    cudaPointerAttributes a;
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
        cudaGetLastError();
        set_last_error(ERR_ARG, "%s: %s is not a device pointer", fn, name);
        return ERR_ARG;
    }
    if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) {
        set_last_error(ERR_ARG, "%s: %s is not a device pointer", fn, name);
        return ERR_ARG;
    }
    int cur = 0;
    if (a.type == cudaMemoryTypeDevice && cudaGetDevice(&cur) == cudaSuccess && a.device != cur) {
        set_last_error(ERR_ARG, "%s: %s is on device %d, the current one is %d", fn, name, a.device, cur);
        return ERR_ARG;
    }
    return OK;
}

}  // namespace cg

using namespace cg;

namespace {

int opt_ptr(const char *fn, const char *name, const void *p) { return p ? dev_ptr(fn, name, p) : OK; }

int rows_shape(const char *fn, long ld, int rows, int vocab) {
    if (rows < 0 || vocab < 1 || ld < vocab) {
        set_last_error(ERR_ARG, "%s: bad shape rows=%d vocab=%d ld=%ld", fn, rows, vocab, ld);
        return ERR_ARG;
    }
    if (vocab > ROW_MAX_VOCAB) {
        set_last_error(ERR_ARG, "%s: vocab %d > %d unsupported", fn, vocab, ROW_MAX_VOCAB);
        return ERR_ARG;
    }
    return OK;
}

}  // namespace

extern "C" int cngpt_cuda_sample(const float *logits, long ld, int rows, int vocab, const float *temperature,
                                 const int *top_k, const float *top_p, const float *min_p, const float *u,
                                 int *tokens, float *logprob) {
    const char *fn = "sample";
    CG_TRY(rows_shape(fn, ld, rows, vocab));
    if (vocab > SAMPLE_MAX_VOCAB) {
        set_last_error(ERR_ARG, "%s: vocab %d > %d unsupported", fn, vocab, SAMPLE_MAX_VOCAB);
        return ERR_ARG;
    }
    if (rows == 0) return OK;
    CG_TRY(dev_ptr(fn, "logits", logits));
    CG_TRY(opt_ptr(fn, "temperature", temperature));
    CG_TRY(opt_ptr(fn, "top_k", top_k));
    CG_TRY(opt_ptr(fn, "top_p", top_p));
    CG_TRY(opt_ptr(fn, "min_p", min_p));
    CG_TRY(dev_ptr(fn, "u", u));
    CG_TRY(dev_ptr(fn, "tokens", tokens));
    CG_TRY(opt_ptr(fn, "logprob", logprob));
    SampleRows a{logits, ld, rows, vocab, temperature, top_k, top_p, min_p, u, tokens, logprob};
    return sample_rows(a, g_stream);
}

extern "C" int cngpt_cuda_topk(const float *logits, long ld, int rows, int vocab, int k, float *values,
                               int *indices) {
    const char *fn = "topk";
    CG_TRY(rows_shape(fn, ld, rows, vocab));
    if (k < 1 || k > vocab || k > TOPK_MAX) {
        set_last_error(ERR_ARG, "%s: k=%d outside [1, min(vocab=%d, %d)]", fn, k, vocab, TOPK_MAX);
        return ERR_ARG;
    }
    if (rows == 0) return OK;
    CG_TRY(dev_ptr(fn, "logits", logits));
    CG_TRY(dev_ptr(fn, "values", values));
    CG_TRY(dev_ptr(fn, "indices", indices));
    return topk_rows(logits, ld, rows, vocab, k, values, indices, g_stream);
}

extern "C" int cngpt_cuda_distill(const float *logits, long ld, int rows, int vocab, const float *top_val,
                                  const int *top_idx, int k, const int *targets, float temperature, float alpha,
                                  float scale, float *loss, float *row_loss, float *dlogits, long ldd) {
    const char *fn = "distill";
    CG_TRY(rows_shape(fn, ld, rows, vocab));
    if (k < 0 || k > TOPK_MAX) {
        set_last_error(ERR_ARG, "%s: k=%d outside [0, %d]", fn, k, TOPK_MAX);
        return ERR_ARG;
    }
    if (!(temperature > 0.0f) || !std::isfinite(temperature) || !(alpha >= 0.0f && alpha <= 1.0f)) {
        set_last_error(ERR_ARG, "%s: temperature %g must be positive and alpha %g in [0, 1]", fn, (double)temperature,
                       (double)alpha);
        return ERR_ARG;
    }
    CG_TRY(dev_ptr(fn, "loss", loss));
    if (rows > 0) {
        CG_TRY(dev_ptr(fn, "logits", logits));
        CG_TRY(dev_ptr(fn, "row_loss", row_loss));
        if (k > 0 && alpha > 0.0f) {
            CG_TRY(dev_ptr(fn, "top_val", top_val));
            CG_TRY(dev_ptr(fn, "top_idx", top_idx));
        }
        if (alpha < 1.0f) CG_TRY(dev_ptr(fn, "targets", targets));
        CG_TRY(opt_ptr(fn, "dlogits", dlogits));
        if (dlogits) {
            const uintptr_t a0 = (uintptr_t)logits, a1 = a0 + ((size_t)(rows - 1) * ld + vocab) * sizeof(float);
            const uintptr_t b0 = (uintptr_t)dlogits, b1 = b0 + ((size_t)(rows - 1) * ldd + vocab) * sizeof(float);
            if (ldd < vocab || (a0 < b1 && b0 < a1 && !(dlogits == logits && (ldd == ld || rows == 1)))) {
                set_last_error(ERR_ARG, "%s: dlogits (pitch %ld) must not overlap logits (pitch %ld) unless both are one",
                               fn, ldd, ld);
                return ERR_ARG;
            }
        }
        CG_TRY(distill_rows(logits, ld, rows, vocab, top_val, top_idx, alpha > 0.0f ? k : 0,
                            alpha < 1.0f ? targets : nullptr, temperature, alpha, scale, row_loss, dlogits, ldd,
                            g_stream));
    }
    return distill_loss_sum(row_loss, rows, scale, loss, g_stream);
}

namespace {
int prefix_shape(int B, int H, int Hk, int hs, int P, int S) {
    if (B < 0 || H < 1 || Hk < 1 || H % Hk != 0 || hs < 1 || hs > 256 || P < 0 || P > (1 << 30) || S < 0 ||
        S > (1 << 30) || (long)B * H > (1L << 30)) {
        set_last_error(ERR_ARG, "prefix_attention: bad shape B=%d n_head=%d n_kv_head=%d hs=%d prefix=%d suffix=%d", B, H,
                       Hk, hs, P, S);
        return ERR_ARG;
    }
    return OK;
}
}  // namespace

extern "C" size_t cngpt_cuda_prefix_attention_workspace(int B, int n_head, int n_kv_head, int hs, int prefix_len,
                                                        int max_suffix) {
    if (prefix_shape(B, n_head, n_kv_head, hs, prefix_len, max_suffix) != OK) return 0;
    return prefix_attention_ws_bytes(B, n_head, n_kv_head, hs, prefix_len, max_suffix);
}

extern "C" int cngpt_cuda_prefix_attention(const float *q, long ldq, const float *pk, const float *pv, long ldp,
                                           int prefix_len, const float *sk, const float *sv, long lds,
                                           long seq_stride, const int *suffix_len, int max_suffix, float *out,
                                           long ldo, int B, int n_head, int n_kv_head, int hs, float scale, void *ws,
                                           size_t ws_bytes) {
    const char *fn = "prefix_attention";
    CG_TRY(prefix_shape(B, n_head, n_kv_head, hs, prefix_len, max_suffix));
    const long row = (long)n_head * hs, kv = (long)n_kv_head * hs;
    if (ldq < row || ldo < row || (prefix_len > 0 && ldp < kv) ||
        (max_suffix > 0 && (lds < kv || (B > 1 && seq_stride < (long)(max_suffix - 1) * lds + kv)))) {
        set_last_error(ERR_ARG, "%s: bad pitch ldq=%ld ldo=%ld ldp=%ld lds=%ld seq_stride=%ld", fn, ldq, ldo, ldp, lds,
                       seq_stride);
        return ERR_ARG;
    }
    if (B == 0) return OK;
    CG_TRY(dev_ptr(fn, "q", q));
    CG_TRY(dev_ptr(fn, "out", out));
    if (prefix_len > 0) {
        CG_TRY(dev_ptr(fn, "pk", pk));
        CG_TRY(dev_ptr(fn, "pv", pv));
    }
    if (max_suffix > 0) {
        CG_TRY(dev_ptr(fn, "sk", sk));
        CG_TRY(dev_ptr(fn, "sv", sv));
        CG_TRY(dev_ptr(fn, "suffix_len", suffix_len));
    }
    const size_t need = prefix_attention_ws_bytes(B, n_head, n_kv_head, hs, prefix_len, max_suffix);
    if (need > 0) {
        CG_TRY(dev_ptr(fn, "ws", ws));
        if (ws_bytes < need || (uintptr_t)ws % 16) {
            set_last_error(ERR_ARG, "%s: the workspace needs %zu bytes at a 16-byte boundary, got %zu at %p", fn, need,
                           ws_bytes, ws);
            return ERR_ARG;
        }
    }
    PrefixAttn a{q, pk, pv, sk, sv, ldq, ldp, lds, seq_stride, ldo, prefix_len, max_suffix, suffix_len, out,
                 B, n_head, n_kv_head, hs, scale};
    return prefix_attention(a, ws, g_stream);
}
