// What the sequence operators of include/hiertcn_ops.h share on the host: version, struct sizes, this thread's error message.
#include <stdarg.h>
#include <stdio.h>

#include "ops.h"

static thread_local char g_ops_err[512] = "";

int ops_fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_ops_err, sizeof(g_ops_err), fmt, ap);
  va_end(ap);
  return code;
}

extern "C" {
int hiertcn_ops_version(void) { return HIERTCN_OPS_VERSION; }
const char* hiertcn_ops_last_error(void) { return g_ops_err; }
int hiertcn_ops_struct_sizes(size_t out[HIERTCN_OPS_N_STRUCTS]) {
  if (!out) return ops_fail(HIERTCN_ERR_INVALID, "null argument");
  const size_t s[HIERTCN_OPS_N_STRUCTS] = {sizeof(hiertcn_glr_t), sizeof(hiertcn_rows_t), sizeof(hiertcn_preference_t), sizeof(hiertcn_policy_t),
                                           sizeof(hiertcn_adamw_tensor_t), sizeof(hiertcn_adamw_t)};
  for (int i = 0; i < HIERTCN_OPS_N_STRUCTS; i++) out[i] = s[i];
  return HIERTCN_OK;
}
}  // extern "C"
