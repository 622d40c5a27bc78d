// The C entry points of gated_ffn: checks and dispatch on the operand type (the products are in policy_ffn_*.cu)
#include "policy_ffn.cuh"

namespace inb {
namespace pol {

static int ffn_check(const InbFfnArgs* p, bool bwd, bool sizes_only) {
  if (p == nullptr) return -1;
  const InbFfnArgs& a = *p;
  if ((a.dtype != INB_BF16 && a.dtype != INB_F16) || (a.act != INB_ACT_SILU && a.act != INB_ACT_GELU) || a.N < 0 ||
      a.N > INB_MAX_FFN || a.D < 1 || a.D > INB_MAX_FFN || a.F < 1 || a.F > INB_MAX_FFN || a.ldh % 8 != 0 || a.ldh < a.F)
    return -2;
  if (a.N == 0) return 0;
  if (a.x == nullptr || a.wg == nullptr || a.wu == nullptr || a.wd == nullptr) return -3;
  if (sizes_only) return 0;
  if (a.h == nullptr || (((uintptr_t)a.h | (uintptr_t)a.g | (uintptr_t)a.u) & 15) != 0) return -3;
  if (!bwd && (a.y == nullptr || (a.g == nullptr) != (a.u == nullptr))) return -3;
  if (bwd && (a.dy == nullptr || a.g == nullptr || a.u == nullptr || (a.dwg == nullptr) != (a.dwu == nullptr) ||
              ((a.dx != nullptr || a.dwg != nullptr) &&
               (a.dg == nullptr || a.du == nullptr || (((uintptr_t)a.dg | (uintptr_t)a.du) & 15) != 0))))
    return -3;
  if (few_rows(a, bwd)) return 0;
  if (a.work_bytes < ffn_work(a, bwd) || (a.work_bytes > 0 && ((uintptr_t)a.work & 15) != 0)) return -5;
  return 0;
}

static int ffn_run(const InbFfnArgs* args, bool bwd, void* stream) {
  const int rc = ffn_check(args, bwd, false);
  if (rc != 0 || args->N == 0) return rc;
  if (few_rows(*args, bwd)) return ffn_rows_any(*args, (cudaStream_t)stream);
  return (args->dtype == INB_BF16 ? ffn_bf16 : ffn_f16)(*args, bwd, (cudaStream_t)stream);
}

}  // namespace pol
}  // namespace inb

extern "C" int inb_gated_ffn_fwd(const InbFfnArgs* args, void* cuda_stream) {
  return inb::pol::ffn_run(args, false, cuda_stream);
}

extern "C" int inb_gated_ffn_bwd(const InbFfnArgs* args, void* cuda_stream) {
  return inb::pol::ffn_run(args, true, cuda_stream);
}

extern "C" int inb_gated_ffn_work(const InbFfnArgs* args, int32_t backward, int64_t* bytes) {
  if (bytes == nullptr) return -1;
  *bytes = 0;
  const int rc = inb::pol::ffn_check(args, backward != 0, true);
  if (rc != 0 || args->N == 0) return rc;
  if (!inb::pol::few_rows(*args, backward != 0)) *bytes = inb::pol::ffn_work(*args, backward != 0);
  return 0;
}
