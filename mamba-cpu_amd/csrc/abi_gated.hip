// C-ABI entry points of the gated linear recurrence: argument checks,
// workspace layout, launches.
#include <climits>
#include <cstring>

#include "abi_util.h"
#include "gated_scan.h"

namespace mcpu {
namespace {

bool any_negative(std::initializer_list<const int64_t*> strides, int n) {
  for (const int64_t* s : strides)
    for (int i = 0; i < n; ++i)
      if (s[i] < 0) return true;
  return false;
}

int64_t chunks_of(const mcpu_gated_scan_args* a, int waves) {
  return (a->seqlen + waves * kGatedT - 1) / (waves * kGatedT);
}

// The kernels reach an element by 32-bit byte offsets, of its channel and its
// step, from a segment's first step; the sum stays below 2^32, where buffer
// accesses end.
bool in_reach(const mcpu_gated_scan_args* a, std::initializer_list<const int64_t*> strides) {
  const int64_t reach = (int64_t{1} << 32) / dtype_size(a->dtype), dim = a->dim > 0 ? a->dim : 1;
  for (const int64_t* s : strides)
    if (s[2] >= reach / dim || s[1] >= reach / kGatedT || dim * s[2] + kGatedT * s[1] >= reach) return false;
  return true;
}

int check_gated(const mcpu_gated_scan_args* a, const char* what) {
  if (a == nullptr) return fail(MCPU_ERR_INVALID, "%s: null argument block", what);
  if (a->batch < 0 || a->seqlen < 0 || a->dim < 0) return fail(MCPU_ERR_INVALID, "%s: negative size", what);
  if (!valid_dtype(a->dtype)) return fail(MCPU_ERR_INVALID, "%s: bad dtype %d", what, a->dtype);
  const int64_t tiles = (a->dim + 63) / 64;
  if (a->batch > INT_MAX || a->seqlen > (int64_t{1} << 40) || tiles > INT_MAX ||
      (tiles > 0 && a->batch > 0 && chunks_of(a, kGatedBwdWaves) > INT_MAX / (tiles * a->batch)))
    return fail(MCPU_ERR_UNSUPPORTED, "%s: batch x seqlen x dim too large", what);
  if ((a->decay == nullptr && a->dim > 0) ||
      ((a->x == nullptr || a->a_gate == nullptr || a->x_gate == nullptr) && a->batch * a->seqlen * a->dim > 0))
    return fail(MCPU_ERR_INVALID, "%s: x, a_gate, x_gate and decay are required", what);
  if (!(a->c >= 0.f)) return fail(MCPU_ERR_INVALID, "%s: c must not be negative", what);
  if (any_negative({a->x_stride, a->a_stride, a->i_stride}, 3))
    return fail(MCPU_ERR_INVALID, "%s: negative stride", what);
  if (!in_reach(a, {a->x_stride, a->a_stride, a->i_stride}))
    return fail(MCPU_ERR_UNSUPPORTED, "%s: a row's steps or channels lie too far apart", what);
  return MCPU_OK;
}

// The tickets and records of a call of more than one chunk.
size_t ticket_bytes(const mcpu_gated_scan_args* a) {
  return align_up(sizeof(uint32_t) * a->batch * ((a->dim + 63) / 64));
}
size_t record_bytes(const mcpu_gated_scan_args* a, int64_t chunks) {
  return chunks > 1 ? ticket_bytes(a) + align_up(sizeof(uint64_t) * a->batch * chunks * a->dim) : 0;
}
int clear_records(GatedScanParams& p, const mcpu_gated_scan_args* a, void* workspace, hipStream_t st) {
  if (p.chunks == 1) return MCPU_OK;
  p.tickets = static_cast<uint32_t*>(workspace);
  p.records = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + ticket_bytes(a));
  return zero_f32(static_cast<float*>(workspace), static_cast<int64_t>(record_bytes(a, p.chunks) / sizeof(float)), st);
}

GatedScanParams make_gated(const mcpu_gated_scan_args* a, int waves) {
  GatedScanParams p;
  std::memset(&p, 0, sizeof(p));
  p.x = a->x;
  p.a_gate = a->a_gate;
  p.x_gate = a->x_gate;
  p.decay = a->decay;
  p.init = a->initial_state;
  p.seq_idx = a->seq_idx;
  p.batch = a->batch;
  p.len = a->seqlen;
  p.dim = a->dim;
  p.c = a->c;
  p.chunks = chunks_of(a, waves);
  p.ckpt = a->ckpt;
  for (int i = 0; i < 3; ++i) {
    p.sx[i] = a->x_stride[i];
    p.sa[i] = a->a_stride[i];
    p.si[i] = a->i_stride[i];
    p.sy[i] = a->y_stride[i];
    p.sdy[i] = a->dy_stride[i];
    p.sdx[i] = a->dx_stride[i];
    p.sda[i] = a->da_stride[i];
    p.sdi[i] = a->di_stride[i];
  }
  return p;
}

}  // namespace
}  // namespace mcpu

using namespace mcpu;

extern "C" size_t mcpu_gated_scan_ckpt_size(const mcpu_gated_scan_args* a) {
  if (check_gated(a, "gated_scan") != MCPU_OK) {
    clear_error();
    return 0;
  }
  return sizeof(float) * a->batch * ((a->seqlen + kGatedT - 1) / kGatedT) * a->dim;
}

extern "C" size_t mcpu_gated_scan_fwd_workspace_size(const mcpu_gated_scan_args* a) {
  if (check_gated(a, "gated_scan") != MCPU_OK) {
    clear_error();
    return 0;
  }
  return record_bytes(a, chunks_of(a, kGatedFwdWaves));
}

extern "C" int mcpu_gated_scan_fwd(const mcpu_gated_scan_args* a, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  const char* what = "gated_scan_fwd";
  clear_error();
  if (int rc = check_gated(a, what)) return rc;
  if (a->y == nullptr && a->batch * a->seqlen * a->dim > 0)
    return fail(MCPU_ERR_INVALID, "%s: y is required", what);
  if (any_negative({a->y_stride}, 3)) return fail(MCPU_ERR_INVALID, "%s: negative stride", what);
  if (!in_reach(a, {a->y_stride}))
    return fail(MCPU_ERR_UNSUPPORTED, "%s: a row's steps or channels lie too far apart", what);
  if (int rc = check_workspace(what, workspace, workspace_bytes, mcpu_gated_scan_fwd_workspace_size(a))) return rc;
  if (int rc = mcpu_check_device()) return rc;
  GatedScanParams p = make_gated(a, kGatedFwdWaves);
  p.y = a->y;
  p.last = a->last_state;
  if (a->batch == 0 || a->dim == 0) return MCPU_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->seqlen == 0)
    return a->last_state == nullptr
               ? MCPU_OK
               : hip_status(gated_edge_launch(a->initial_state, a->last_state, a->batch * a->dim, st), what);
  if (int rc = clear_records(p, a, workspace, st)) return rc;
  return hip_status(gated_scan_fwd_launch(p, a->dtype, st), "gated_scan_fwd launch");
}

extern "C" size_t mcpu_gated_scan_bwd_workspace_size(const mcpu_gated_scan_args* a) {
  if (check_gated(a, "gated_scan") != MCPU_OK) {
    clear_error();
    return 0;
  }
  const int64_t chunks = chunks_of(a, kGatedBwdWaves);
  return record_bytes(a, chunks) + align_up(sizeof(float) * a->batch * chunks * a->dim);
}

extern "C" int mcpu_gated_scan_bwd(const mcpu_gated_scan_args* a, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  const char* what = "gated_scan_bwd";
  clear_error();
  if (int rc = check_gated(a, what)) return rc;
  const int64_t n = a->batch * a->seqlen * a->dim;
  if ((n > 0 && (a->dy == nullptr || a->dx == nullptr || a->da_gate == nullptr || a->dx_gate == nullptr)) ||
      (a->dim > 0 && a->ddecay == nullptr))
    return fail(MCPU_ERR_INVALID, "%s: dy, dx, da_gate, dx_gate and ddecay are required", what);
  if (n > 0 && a->ckpt == nullptr)
    return fail(MCPU_ERR_INVALID, "%s: the states the forward kept (ckpt) are required", what);
  if (any_negative({a->dy_stride, a->dx_stride, a->da_stride, a->di_stride}, 3))
    return fail(MCPU_ERR_INVALID, "%s: negative stride", what);
  if (!in_reach(a, {a->dy_stride, a->dx_stride, a->da_stride, a->di_stride}))
    return fail(MCPU_ERR_UNSUPPORTED, "%s: a row's steps or channels lie too far apart", what);
  if (int rc = check_workspace(what, workspace, workspace_bytes, mcpu_gated_scan_bwd_workspace_size(a))) return rc;
  if (int rc = mcpu_check_device()) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->dim == 0) return MCPU_OK;
  if (a->batch == 0 || a->seqlen == 0) {
    if (int rc = zero_f32(a->ddecay, a->dim, st)) return rc;
    return a->batch == 0 || a->dinitial_state == nullptr
               ? MCPU_OK
               : hip_status(gated_edge_launch(a->dlast_state, a->dinitial_state, a->batch * a->dim, st), what);
  }
  GatedScanParams p = make_gated(a, kGatedBwdWaves);
  p.dy = a->dy;
  p.dlast = a->dlast_state;
  p.dx = a->dx;
  p.da_gate = a->da_gate;
  p.dx_gate = a->dx_gate;
  p.ddecay = a->ddecay;
  p.dinit = a->dinitial_state;
  p.ddecay_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + record_bytes(a, p.chunks));
  if (int rc = clear_records(p, a, workspace, st)) return rc;
  return hip_status(gated_scan_bwd_launch(p, a->dtype, st), "gated_scan_bwd launch");
}

extern "C" int mcpu_gated_step(const mcpu_gated_step_args* a, void* stream) {
  const char* what = "gated_step";
  clear_error();
  if (a == nullptr) return fail(MCPU_ERR_INVALID, "%s: null argument block", what);
  if (a->batch < 0 || a->dim < 0 || a->state_batch < 0) return fail(MCPU_ERR_INVALID, "%s: negative size", what);
  if (!valid_dtype(a->dtype)) return fail(MCPU_ERR_INVALID, "%s: bad dtype %d", what, a->dtype);
  if (!(a->c >= 0.f)) return fail(MCPU_ERR_INVALID, "%s: c must not be negative", what);
  if (a->dim > 0 && a->batch > (int64_t{1} << 38) / a->dim)
    return fail(MCPU_ERR_UNSUPPORTED, "%s: batch x dim too large", what);
  if (a->batch * a->dim > 0 && (a->x == nullptr || a->a_gate == nullptr || a->x_gate == nullptr ||
                                a->decay == nullptr || a->y == nullptr ||
                                (a->state == nullptr && a->state_batch > 0)))
    return fail(MCPU_ERR_INVALID, "%s: state, x, a_gate, x_gate, decay and y are required", what);
  if (a->state_batch_indices == nullptr && a->state_batch < a->batch)
    return fail(MCPU_ERR_INVALID, "%s: state has fewer rows than the batch", what);
  if (any_negative({a->state_stride, a->x_stride, a->a_stride, a->i_stride}, 2))
    return fail(MCPU_ERR_INVALID, "%s: negative stride", what);
  if (int rc = mcpu_check_device()) return rc;
  if (a->batch == 0 || a->dim == 0) return MCPU_OK;
  GatedStepParams p;
  std::memset(&p, 0, sizeof(p));
  p.state = a->state;
  p.x = a->x;
  p.a_gate = a->a_gate;
  p.x_gate = a->x_gate;
  p.decay = a->decay;
  p.y = a->y;
  p.batch = a->batch;
  p.dim = a->dim;
  p.c = a->c;
  for (int i = 0; i < 2; ++i) {
    p.sst[i] = a->state_stride[i];
    p.sx[i] = a->x_stride[i];
    p.sa[i] = a->a_stride[i];
    p.si[i] = a->i_stride[i];
  }
  p.state_idx = a->state_batch_indices;
  p.state_batch = a->state_batch;
  return hip_status(gated_step_launch(p, a->dtype, static_cast<hipStream_t>(stream)), "gated_step launch");
}
