// C-ABI entry points of the residual norm, the embedding and the token sampler:
// argument checks, workspace layout, launches.
#include <climits>
#include <cstring>

#include "abi_util.h"
#include "lm_params.h"

namespace mcpu {
namespace {

// ---- residual norm ----------------------------------------------------------------

int check_norm(const mcpu_norm_args* a, const char* what) {
  if (a == nullptr) return fail(MCPU_ERR_INVALID, "%s: null argument block", what);
  if (a->rows < 0 || a->dim < 0) return fail(MCPU_ERR_INVALID, "%s: negative size", what);
  if (!valid_dtype(a->dtype) || (a->res_dtype != a->dtype && a->res_dtype != MCPU_F32))
    return fail(MCPU_ERR_INVALID, "%s: bad dtype %d with residual dtype %d", what, a->dtype, a->res_dtype);
  if (a->rms != 0 && a->rms != 1) return fail(MCPU_ERR_INVALID, "%s: rms must be 0 or 1", what);
  if (!(a->eps >= 0.f)) return fail(MCPU_ERR_INVALID, "%s: eps must not be negative", what);
  if (a->rows > INT_MAX || a->dim > (int64_t{1} << 24))
    return fail(MCPU_ERR_UNSUPPORTED, "%s: at most 2^31 - 1 rows of 2^24 elements", what);
  if ((a->weight == nullptr && a->dim > 0) || (a->x == nullptr && a->z == nullptr && a->rows * a->dim > 0))
    return fail(MCPU_ERR_INVALID, "%s: x (or z) and weight are required", what);
  if (a->x_stride < 0 || a->res_stride < 0 || a->y_stride < 0 || a->dy_stride < 0)
    return fail(MCPU_ERR_INVALID, "%s: negative stride", what);
  return MCPU_OK;
}

NormParams make_norm(const mcpu_norm_args* a) {
  NormParams p;
  std::memset(&p, 0, sizeof(p));
  p.x = a->x;
  p.residual = a->residual;
  p.weight = a->weight;
  p.bias = a->bias;
  p.rows = a->rows;
  p.dim = a->dim;
  p.sx = a->x_stride;
  p.sres = a->res_stride;
  p.sy = a->y_stride;
  p.sdy = a->dy_stride;
  p.eps = a->eps;
  p.rms = a->rms;
  p.x_dtype = a->dtype;
  p.res_dtype = a->res_dtype;
  p.mean = a->mean;
  p.rstd = a->rstd;
  return p;
}

// ---- embedding ----------------------------------------------------------------------

int check_embedding(const mcpu_embedding_args* a, const char* what) {
  if (a == nullptr) return fail(MCPU_ERR_INVALID, "%s: null argument block", what);
  if (a->tokens < 0 || a->vocab < 0 || a->dim < 0) return fail(MCPU_ERR_INVALID, "%s: negative size", what);
  if (!valid_dtype(a->dtype) || (a->ids64 != 0 && a->ids64 != 1))
    return fail(MCPU_ERR_INVALID, "%s: bad dtype %d or ids64 %d", what, a->dtype, a->ids64);
  if (a->weight_stride < 0 || a->dout_stride < 0) return fail(MCPU_ERR_INVALID, "%s: negative stride", what);
  if (a->tokens > INT_MAX - 64 || a->vocab > INT_MAX - 1024 || a->dim > INT_MAX)
    return fail(MCPU_ERR_UNSUPPORTED, "%s: tokens, vocab and dim must fit 31 bits", what);
  if (embedding_chunks(a->tokens) * ((a->dim + 1023) / 1024) + a->vocab / 16 > INT_MAX - 1)
    return fail(MCPU_ERR_UNSUPPORTED, "%s: tokens x dim too large", what);
  if (a->tokens > 0 && a->ids == nullptr) return fail(MCPU_ERR_INVALID, "%s: ids are required", what);
  return MCPU_OK;
}

EmbeddingParams make_embedding(const mcpu_embedding_args* a) {
  EmbeddingParams p;
  std::memset(&p, 0, sizeof(p));
  p.ids = a->ids;
  p.ids64 = a->ids64;
  p.weight = a->weight;
  p.tokens = a->tokens;
  p.vocab = a->vocab;
  p.dim = a->dim;
  p.sw = a->weight_stride;
  p.sdo = a->dout_stride;
  p.scale = a->scale;
  p.dtype = a->dtype;
  return p;
}

// ---- sampling -----------------------------------------------------------------------

int check_sample(const mcpu_sample_args* a, const char* what) {
  if (a == nullptr) return fail(MCPU_ERR_INVALID, "%s: null argument block", what);
  if (a->rows < 0 || a->vocab < 0) return fail(MCPU_ERR_INVALID, "%s: negative size", what);
  if (!valid_dtype(a->dtype)) return fail(MCPU_ERR_INVALID, "%s: bad dtype %d", what, a->dtype);
  if (a->logits_stride < 0 || a->noise_stride < 0) return fail(MCPU_ERR_INVALID, "%s: negative stride", what);
  if (a->rows > INT_MAX || a->vocab > (1 << 23))
    return fail(MCPU_ERR_UNSUPPORTED, "%s: at most 2^31 - 1 rows of 2^23 logits", what);
  if (a->rows > 0 && a->vocab == 0) return fail(MCPU_ERR_INVALID, "%s: no logits to choose from", what);
  if (a->temperature_rows == nullptr && !(a->temperature == a->temperature))
    return fail(MCPU_ERR_INVALID, "%s: temperature must be a number", what);
  if (a->top_p_rows == nullptr && !(a->top_p >= 0.f && a->top_p <= 1.f))
    return fail(MCPU_ERR_INVALID, "%s: top_p must lie in [0, 1]", what);
  if (a->min_p_rows == nullptr && !(a->min_p >= 0.f && a->min_p <= 1.f))
    return fail(MCPU_ERR_INVALID, "%s: min_p must lie in [0, 1]", what);
  if (a->top_k_rows == nullptr && a->top_k < 0) return fail(MCPU_ERR_INVALID, "%s: top_k must not be negative", what);
  const bool greedy = a->temperature_rows == nullptr && a->temperature <= 0.f;
  if (a->rows > 0 && (a->logits == nullptr || a->token == nullptr || (a->noise == nullptr && !greedy)))
    return fail(MCPU_ERR_INVALID, "%s: logits, token and noise (above temperature 0) are required", what);
  return MCPU_OK;
}

SampleParams make_sample(const mcpu_sample_args* a) {
  SampleParams p;
  std::memset(&p, 0, sizeof(p));
  p.logits = a->logits;
  p.noise = a->noise;
  p.temperature = a->temperature;
  p.top_p = a->top_p;
  p.min_p = a->min_p;
  p.top_k = a->top_k;
  p.temperature_rows = a->temperature_rows;
  p.top_p_rows = a->top_p_rows;
  p.min_p_rows = a->min_p_rows;
  p.top_k_rows = a->top_k_rows;
  p.token = a->token;
  p.logprob = a->logprob;
  p.rows = a->rows;
  p.vocab = a->vocab;
  p.sl = a->logits_stride;
  p.sn = a->noise_stride;
  p.dtype = a->dtype;
  return p;
}

}  // namespace
}  // namespace mcpu

using namespace mcpu;

extern "C" int mcpu_norm_fwd(const mcpu_norm_args* a, void* stream) {
  const char* what = "norm_fwd";
  clear_error();
  if (int rc = check_norm(a, what)) return rc;
  if ((a->y == nullptr || a->x == nullptr) && a->rows * a->dim > 0)
    return fail(MCPU_ERR_INVALID, "%s: x and y are required", what);
  if (int rc = mcpu_check_device()) return rc;
  if (a->rows == 0 || a->dim == 0) return MCPU_OK;
  NormParams p = make_norm(a);
  p.y = a->y;
  p.res_out = a->res_out;
  return hip_status(norm_fwd_launch(p, static_cast<hipStream_t>(stream)), "norm_fwd launch");
}

extern "C" size_t mcpu_norm_bwd_workspace_size(const mcpu_norm_args* a) {
  if (check_norm(a, "norm") != MCPU_OK) {
    clear_error();
    return 0;
  }
  return align_up(sizeof(float) * 2 * norm_bwd_parts(a->rows, a->dim) * a->dim);
}

extern "C" int mcpu_norm_bwd(const mcpu_norm_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "norm_bwd";
  clear_error();
  if (int rc = check_norm(a, what)) return rc;
  const int64_t n = a->rows * a->dim;
  if ((n > 0 && (a->dy == nullptr || a->dx == nullptr || a->rstd == nullptr || (!a->rms && a->mean == nullptr))) ||
      (a->dim > 0 && (a->dweight == nullptr || (a->bias != nullptr && a->dbias == nullptr))))
    return fail(MCPU_ERR_INVALID, "%s: dy, rstd, mean (layer norm), dx, dweight and dbias (with a bias) are required",
                what);
  if (int rc = check_workspace(what, workspace, workspace_bytes, mcpu_norm_bwd_workspace_size(a))) return rc;
  if (int rc = mcpu_check_device()) return rc;
  if (a->dim == 0) return MCPU_OK;
  NormParams p = make_norm(a);
  p.z = a->z;
  p.dy = a->dy;
  p.dres_out = a->dres_out;
  p.dx = a->dx;
  p.dres = a->dres;
  p.dweight = a->dweight;
  p.dbias = a->bias != nullptr ? a->dbias : nullptr;
  p.part = static_cast<float*>(workspace);
  p.parts = norm_bwd_parts(a->rows, a->dim);
  return hip_status(norm_bwd_launch(p, static_cast<hipStream_t>(stream)), "norm_bwd launch");
}

extern "C" int mcpu_embedding_fwd(const mcpu_embedding_args* a, void* stream) {
  const char* what = "embedding_fwd";
  clear_error();
  if (int rc = check_embedding(a, what)) return rc;
  if (a->tokens * a->dim > 0 && ((a->weight == nullptr && a->vocab > 0) || a->out == nullptr))
    return fail(MCPU_ERR_INVALID, "%s: weight and out are required", what);
  if (int rc = mcpu_check_device()) return rc;
  if (a->tokens == 0 || a->dim == 0) return MCPU_OK;
  EmbeddingParams p = make_embedding(a);
  p.out = a->out;
  return hip_status(embedding_fwd_launch(p, static_cast<hipStream_t>(stream)), "embedding_fwd launch");
}

extern "C" size_t mcpu_embedding_bwd_workspace_size(const mcpu_embedding_args* a) {
  if (check_embedding(a, "embedding") != MCPU_OK) {
    clear_error();
    return 0;
  }
  return align_up(sizeof(int32_t) * a->tokens) + align_up(sizeof(int32_t) * (a->vocab + 1)) +
         align_up(sizeof(float) * 2 * embedding_chunks(a->tokens) * a->dim);
}

extern "C" int mcpu_embedding_bwd(const mcpu_embedding_args* a, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  const char* what = "embedding_bwd";
  clear_error();
  if (int rc = check_embedding(a, what)) return rc;
  if ((a->tokens * a->dim > 0 && a->dout == nullptr) || (a->vocab * a->dim > 0 && a->dweight == nullptr))
    return fail(MCPU_ERR_INVALID, "%s: dout and dweight are required", what);
  if (a->dim > 65535 * 256) return fail(MCPU_ERR_UNSUPPORTED, "%s: at most 65535 x 256 columns", what);
  if (int rc = check_workspace(what, workspace, workspace_bytes, mcpu_embedding_bwd_workspace_size(a))) return rc;
  if (int rc = mcpu_check_device()) return rc;
  if (a->vocab == 0 || a->dim == 0) return MCPU_OK;
  EmbeddingParams p = make_embedding(a);
  p.dout = a->dout;
  p.dweight = a->dweight;
  char* ws = static_cast<char*>(workspace);
  p.order = reinterpret_cast<int32_t*>(ws);
  ws += align_up(sizeof(int32_t) * a->tokens);
  p.start = reinterpret_cast<int32_t*>(ws);
  ws += align_up(sizeof(int32_t) * (a->vocab + 1));
  p.part = reinterpret_cast<float*>(ws);
  return hip_status(embedding_bwd_launch(p, static_cast<hipStream_t>(stream)), "embedding_bwd launch");
}

extern "C" size_t mcpu_sample_workspace_size(const mcpu_sample_args* a) {
  if (check_sample(a, "sample") != MCPU_OK) {
    clear_error();
    return 0;
  }
  return align_up(sample_workspace(make_sample(a)));
}

extern "C" int mcpu_sample(const mcpu_sample_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "sample";
  clear_error();
  if (int rc = check_sample(a, what)) return rc;
  if (int rc = check_workspace(what, workspace, workspace_bytes, mcpu_sample_workspace_size(a))) return rc;
  if (int rc = mcpu_check_device()) return rc;
  if (a->rows == 0) return MCPU_OK;
  SampleParams p = make_sample(a);
  p.slices = workspace;
  return hip_status(sample_launch(p, static_cast<hipStream_t>(stream)), "sample launch");
}
