// C-ABI entry points of the head's losses: argument checks, workspace layout,
// launches.
#include <cstring>

#include "abi_util.h"
#include "loss_params.h"

namespace mcpu {
namespace {

bool distil(const mcpu_linear_loss_args* a) { return a->teacher != nullptr || a->share != nullptr; }

int check_loss(const mcpu_linear_loss_args* a, const char* what) {
  if (a == nullptr) return fail(MCPU_ERR_INVALID, "%s: null argument block", what);
  if (a->tokens < 0 || a->vocab < 0 || a->dim < 0 || a->k < 0 || a->hidden_stride < 0 || a->weight_stride < 0)
    return fail(MCPU_ERR_INVALID, "%s: negative size or stride", what);
  if (!valid_dtype(a->dtype) || (a->ids64 != 0 && a->ids64 != 1))
    return fail(MCPU_ERR_INVALID, "%s: bad dtype %d or ids64 %d", what, a->dtype, a->ids64);
  if (a->reduction < MCPU_REDUCE_NONE || a->reduction > MCPU_REDUCE_MEAN)
    return fail(MCPU_ERR_INVALID, "%s: bad reduction %d", what, a->reduction);
  if (a->dim == 0) return fail(MCPU_ERR_INVALID, "%s: dim must be positive", what);
  // So that float32 has its inverse times a logit, and its square times a divergence.
  if (!(a->temperature >= 0x1p-60f) || !(a->temperature <= 0x1p60f))
    return fail(MCPU_ERR_INVALID, "%s: temperature must lie in 2^-60 to 2^60", what);
  // Without tokens a teacher's logits have no address to tell by.
  if (!distil(a) && a->tokens > 0 && a->k > 0 && (a->k != 1 || a->temperature != 1.f))
    return fail(MCPU_ERR_INVALID, "%s: cross entropy has one target a row and temperature 1", what);
  if (distil(a) && a->dlse != nullptr) return fail(MCPU_ERR_INVALID, "%s: distillation has no dlse", what);
  if (a->tokens > (1 << 26) || a->vocab > (1 << 24) || a->dim > (1 << 20) || a->k > kLossMaxK)
    return fail(MCPU_ERR_UNSUPPORTED, "%s: at most 2^26 tokens, 2^24 vocabulary rows, 2^20 columns and %lld entries",
                what, static_cast<long long>(kLossMaxK));
  if (a->tokens > 0 && (a->hidden == nullptr || (a->vocab > 0 && a->weight == nullptr) ||
                        (a->k > 0 && (a->ids == nullptr || (distil(a) && a->picked == nullptr))) ||
                        a->stat == nullptr || a->rows == nullptr))
    return fail(MCPU_ERR_INVALID, "%s: hidden, weight, ids, stat, rows and (distillation) picked are required", what);
  return MCPU_OK;
}

// Nothing to take a loss of: no rows, no vocabulary or no entries.
bool nothing(const mcpu_linear_loss_args* a) { return a->tokens == 0 || a->vocab == 0 || a->k == 0; }

// Rows that begin at multiples of 16 bytes.
bool aligned_rows(const void* p, int64_t stride, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * dtype_size(dtype) % 16 == 0;
}

LossParams make_loss(const mcpu_linear_loss_args* a) {
  LossParams p;
  std::memset(&p, 0, sizeof(p));
  p.hidden = a->hidden;
  p.weight = a->weight;
  p.ids = a->ids;
  p.teacher = a->teacher;
  p.ids64 = a->ids64;
  p.tokens = a->tokens;
  p.vocab = a->vocab;
  p.dim = a->dim;
  p.k = a->k;
  p.sh = a->hidden_stride;
  p.sw = a->weight_stride;
  p.ignore = a->ignore_index;
  p.temperature = a->temperature;
  p.dtype = a->dtype;
  p.reduction = a->reduction;
  p.loss = a->loss;
  p.lse = a->lse;
  p.picked = a->picked;
  p.stat = a->stat;
  p.share = a->share;
  p.rows = a->rows;
  p.dloss = a->dloss;
  p.dlse = a->dlse;
  p.dhidden = a->dhidden;
  p.dweight = a->dweight;
  p.few_lds = aligned_rows(a->hidden, a->hidden_stride, a->dtype) &&
              aligned_rows(a->weight, a->weight_stride, a->dtype);
  loss_plan(p);
  return p;
}

// The products read 16-byte groups of whole depths: weight as it lies where it has them.
bool weight_in_place(const mcpu_linear_loss_args* a) {
  return a->dtype != MCPU_F32 && a->dim % kLossDepth == 0 && a->weight_stride <= (int64_t{1} << 20) &&
         aligned_rows(a->weight, a->weight_stride, a->dtype);
}

// Takes parts of a workspace one after the other; without one it counts.
struct Layout {
  char* at;
  size_t used = 0;
  template <typename T> void take(T*& p, int64_t count, size_t each = sizeof(T)) {
    p = at != nullptr ? reinterpret_cast<T*>(at + used) : nullptr;
    used += align_up(static_cast<size_t>(count) * each);
  }
  void take(void*& p, int64_t count, size_t each) {
    char* q;
    take<char>(q, count, each);
    p = q;
  }
};

// Weight as the forward lays it out, behind its largest magnitude; none where it is read in place.
size_t laid_bytes(const mcpu_linear_loss_args* a, const LossParams& p) {
  if (weight_in_place(a) || p.blocks) return 0;
  return 256 + align_up(static_cast<size_t>(loss_pieces(a->dtype) * p.vocab * p.dpad) * 2);
}

void lay_operands(const mcpu_linear_loss_args* a, LossParams& p, Layout& w) {
  const int pieces = loss_pieces(a->dtype);
  w.take(p.scal, 1);
  if (!distil(a)) w.take(p.target, p.tpad);
  w.take(p.hrows, pieces * p.tpad * p.dpad, 2);
  if (weight_in_place(a)) return;
  if (a->laid != nullptr && laid_bytes(a, p) > 0) {
    p.laid = static_cast<uint32_t*>(a->laid);
    p.wrows = static_cast<char*>(a->laid) + 256;
  } else {
    w.take(p.wrows, pieces * p.vocab * p.dpad, 2);
  }
}

size_t lay_fwd(const mcpu_linear_loss_args* a, LossParams& p, void* workspace) {
  Layout w{static_cast<char*>(workspace)};
  p.each = p.loss;
  if (p.reduction != MCPU_REDUCE_NONE) w.take(p.each, p.tokens);
  if (distil(a)) w.take(p.keep, p.tokens);
  if (distil(a)) w.take(p.cross, p.tokens);
  if (!distil(a)) w.take(p.picked, p.tpad);
  if (p.tokens <= kLossFew) {
    w.take(p.part, (p.vocab + kLossPart - 1) / kLossPart * kLossFew);
    return w.used;
  }
  if (p.blocks)
    w.take(p.scal, 1);
  else
    lay_operands(a, p, w);
  w.take(p.part, (p.vocab + kLossPart - 1) / kLossPart * p.tpad);
  return w.used;
}

size_t lay_bwd(const mcpu_linear_loss_args* a, LossParams& p, void* workspace) {
  Layout w{static_cast<char*>(workspace)};
  lay_operands(a, p, w);
  w.take(p.coef, 4 * p.tpad);
  // Distillation: rows have units of their own in f16 pieces, where each has a gradient of its own.
  if (!distil(a) || (a->reduction == MCPU_REDUCE_NONE && a->dtype != MCPU_BF16))
    w.take(p.hscaled, loss_pieces(a->dtype) * p.tpad * p.dpad, 2);
  w.take(p.grad, loss_pieces(a->dtype) * p.tpad * p.vpiece, 2);
  if (p.dhidden != nullptr) w.take(p.acc, p.htiles * kLossTile * kLossTile);
  if (p.dweight != nullptr && p.wsplit > 1) w.take(p.dwpart, p.wsplit * p.vpiece * p.dpad);
  return w.used;
}

}  // namespace
}  // namespace mcpu

using namespace mcpu;

extern "C" size_t mcpu_linear_loss_laid_size(const mcpu_linear_loss_args* a) {
  if (check_loss(a, "linear_loss") != MCPU_OK) {
    clear_error();
    return 0;
  }
  return nothing(a) ? 0 : laid_bytes(a, make_loss(a));
}

extern "C" size_t mcpu_linear_loss_fwd_workspace_size(const mcpu_linear_loss_args* a) {
  if (check_loss(a, "linear_loss") != MCPU_OK) {
    clear_error();
    return 0;
  }
  if (nothing(a)) return 0;
  LossParams p = make_loss(a);
  return lay_fwd(a, p, nullptr);
}

extern "C" int mcpu_linear_loss_fwd(const mcpu_linear_loss_args* a, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  const char* what = "linear_loss_fwd";
  clear_error();
  if (int rc = check_loss(a, what)) return rc;
  const int64_t losses = a->reduction == MCPU_REDUCE_NONE ? a->tokens : 1;
  if ((a->loss == nullptr && losses > 0) || (a->tokens > 0 && a->lse == nullptr) ||
      (!nothing(a) && (a->teacher == nullptr) != (a->share == nullptr)))
    return fail(MCPU_ERR_INVALID, "%s: loss, lse, and share with a teacher, are required", what);
  if (int rc = check_workspace(what, workspace, workspace_bytes, mcpu_linear_loss_fwd_workspace_size(a))) return rc;
  if (int rc = mcpu_check_device()) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (nothing(a)) {  // no row counts
    hipError_t e = loss_zero(a->loss, 4 * losses, st);
    if (e == hipSuccess) e = loss_zero(a->lse, 4 * a->tokens, st);
    if (e == hipSuccess) e = loss_zero(a->rows, a->rows != nullptr ? 4 * (a->tokens + 1) : 0, st);
    return hip_status(e, "linear_loss_fwd launch");
  }
  LossParams p = make_loss(a);
  lay_fwd(a, p, workspace);
  return hip_status(loss_fwd_launch(p, st), "linear_loss_fwd launch");
}

extern "C" size_t mcpu_linear_loss_bwd_workspace_size(const mcpu_linear_loss_args* a) {
  if (check_loss(a, "linear_loss") != MCPU_OK) {
    clear_error();
    return 0;
  }
  if (nothing(a)) return 0;
  LossParams p = make_loss(a);
  return lay_bwd(a, p, nullptr);
}

extern "C" int mcpu_linear_loss_bwd(const mcpu_linear_loss_args* a, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  const char* what = "linear_loss_bwd";
  clear_error();
  if (int rc = check_loss(a, what)) return rc;
  if (a->dloss == nullptr && a->reduction != MCPU_REDUCE_NONE)
    return fail(MCPU_ERR_INVALID, "%s: dloss is required where the loss is reduced", what);
  if (int rc = check_workspace(what, workspace, workspace_bytes, mcpu_linear_loss_bwd_workspace_size(a))) return rc;
  if (int rc = mcpu_check_device()) return rc;
  if (a->dhidden == nullptr && a->dweight == nullptr) return MCPU_OK;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (nothing(a)) {
    const int64_t row = a->dim * dtype_size(a->dtype);
    hipError_t e = loss_zero(a->dhidden, a->dhidden != nullptr ? a->tokens * row : 0, st);
    if (e == hipSuccess) e = loss_zero(a->dweight, a->dweight != nullptr ? a->vocab * row : 0, st);
    return hip_status(e, "linear_loss_bwd launch");
  }
  LossParams p = make_loss(a);
  lay_bwd(a, p, workspace);
  return hip_status(loss_bwd_launch(p, st), "linear_loss_bwd launch");
}
