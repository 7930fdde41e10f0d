// ccb_nn_block_norm_backward and its workspace; the kernels are in nn_norm_back.cuh.
#include "nn_norm_back.cuh"

using namespace ccb_nn;

extern "C" int ccb_nn_block_norm_backward_workspace(long long rows, long long cols, size_t* bytes) {
  static const char* const me = "ccb_nn_block_norm_backward_workspace";
  CCB_NN_GUARD(me, {
    if (!bytes) return fail(CCB_ERR_INVALID, me, "null pointer");
    if (rows < 0 || cols < 0 || rows > INT_MAX || cols > (1 << 24)) return fail(CCB_ERR_INVALID, me, "rows must be in [0, 2^31), cols in [0, 2^24]");
    *bytes = back_bytes(rows, cols);
    return CCB_OK;
  })
}

extern "C" int ccb_nn_block_norm_backward(const ccb_nn_block_norm_backward_t* a, void* stream) {
  static const char* const me = "ccb_nn_block_norm_backward";
  CCB_NN_GUARD(me, {
    if (!a) return fail(CCB_ERR_INVALID, me, "null argument block");
    std::string bad = check_common(a->rows, a->cols, a->dtype, a->x_dtype, a->gate_dtype, a->weight_dtype, a->kind, a->act, a->p, a->eps,
                                   a->scale, a->gate != nullptr, a->pre_weight || a->post_weight || a->post_bias);
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    const int tb = type_bytes(a->dtype), xb = type_bytes(a->x_dtype), wb = type_bytes(a->weight_dtype), gb = a->gate ? type_bytes(a->gate_dtype) : 4;
    const bool channel = a->gate && a->gate_stride == 0;
    bad = check_mats(a->rows, a->cols,
                     {{a->y, a->y_stride, xb, "y"}, {a->dy, a->dy_stride, xb, "dy"}, {a->dh, a->dh_stride, tb, "dh"},
                      {a->branch, a->branch_stride, tb, "branch"}, {a->dx, a->dx_stride, xb, "dx"}, {a->dbranch, a->dbranch_stride, tb, "dbranch"},
                      {a->gate, channel ? a->cols : a->gate_stride, gb, "gate"}, {a->dgate, channel ? a->cols : a->dgate_stride, channel ? 4 : gb, "dgate"},
                      {a->pre_weight, a->cols, wb, "pre_weight"}, {a->post_weight, a->cols, wb, "post_weight"},
                      {a->post_bias, a->cols, wb, "post_bias"}, {a->dpre_weight, a->cols, 4, "dpre_weight"}, {a->dpre_bias, a->cols, 4, "dpre_bias"},
                      {a->dpost_weight, a->cols, 4, "dpost_weight"}, {a->dpost_bias, a->cols, 4, "dpost_bias"}});
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    if (a->cols == 0) return CCB_OK;
    const bool sums = a->dpre_weight || a->dpre_bias || a->dpost_weight || a->dpost_bias || (channel && a->dgate);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->rows == 0) {  // sums over no rows
      for (void* v : {a->dpre_weight, a->dpre_bias, a->dpost_weight, a->dpost_bias, channel ? a->dgate : nullptr})
        if (v) {
          const cudaError_t e = cudaMemsetAsync(v, 0, (size_t)a->cols * 4, st);
          if (e != cudaSuccess) return fail(CCB_ERR_DRIVER, me, std::string("cudaMemsetAsync: ") + cudaGetErrorString(e));
        }
      return CCB_OK;
    }
    if (bad.empty() && !a->branch && (a->dbranch || a->gate || a->dgate || a->post_weight || a->post_bias || a->dpost_weight || a->dpost_bias))
      bad = "without a branch there is no gate, post_weight, post_bias or gradient of them";
    if (bad.empty() && a->dgate && !a->gate) bad = "dgate needs the gate";
    if (bad.empty() && !a->post_norm && (a->post_weight || a->post_bias || a->dpost_weight || a->dpost_bias)) bad = "post_weight and post_bias need post_norm";
    if (bad.empty() && !a->dh && (a->pre_weight || a->dpre_weight || a->dpre_bias)) bad = "pre_weight, dpre_weight and dpre_bias need dh";
    if (!bad.empty()) return fail(CCB_ERR_INVALID, me, bad);
    if (!a->y && a->dh) return fail(CCB_ERR_INVALID, me, "null pointer: y");
    if (!a->dy && !a->dh) return fail(CCB_ERR_INVALID, me, "neither dy nor dh is given");
    if (a->base > ~0ull - (u64)a->rows * (u64)a->cols) return fail(CCB_ERR_INVALID, me, "base + rows * cols passes 2^64");
    if (sums && (!a->workspace || a->workspace_bytes < back_bytes(a->rows, a->cols) || !aligned(a->workspace, 16)))
      return fail(CCB_ERR_INVALID, me, "workspace of " + std::to_string(a->workspace_bytes) + " bytes: " + std::to_string(back_bytes(a->rows, a->cols)) +
                                           " are needed, 16-byte aligned");
    int sms = 0;
    if (const int rc = sm_count(me, &sms)) return rc;
    const BackP p = {a->y, a->dy, a->dh, a->branch, a->gate, a->pre_weight, a->post_weight, a->post_bias, a->dx, a->dbranch,
                     channel ? nullptr : a->dgate,
                     {(float*)a->dpre_weight, (float*)a->dpre_bias, (float*)a->dpost_weight, (float*)a->dpost_bias, channel ? (float*)a->dgate : nullptr},
                     (float*)a->workspace, a->rows, a->cols, a->y_stride, a->dy_stride, a->dh_stride, a->branch_stride, a->gate_stride, a->dx_stride,
                     a->dbranch_stride, a->dgate_stride, (float)a->eps, (float)a->scale, a->gate_dtype, a->weight_dtype, a->act, a->post_norm,
                     make_drop(a->p, a->seed, a->offset, a->base, (u64)a->rows * (u64)a->cols)};
    if (a->dtype == CCB_F16)
      backward_f16(a->x_dtype, a->kind, p, sms, st);
    else
      by_type_but_f16<Backward>(a->dtype, a->x_dtype, a->kind, p, sms, st);
    return launched(me);
  })
}
