// C-ABI entry points of the residual norm: argument checks, workspace layout,
// launches.
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
  if ((a->weight == nullptr && a->dim > 0) || (a->x == nullptr && a->rows * a->dim > 0))
    return fail(MCPU_ERR_INVALID, "%s: x and weight are required", what);
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

}  // namespace
}  // namespace mcpu

using namespace mcpu;

extern "C" int mcpu_norm_fwd(const mcpu_norm_args* a, void* stream) {
  const char* what = "norm_fwd";
  clear_error();
  if (int rc = check_norm(a, what)) return rc;
  if (a->y == nullptr && a->rows * a->dim > 0) return fail(MCPU_ERR_INVALID, "%s: y is required", what);
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
