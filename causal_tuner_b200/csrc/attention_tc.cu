#include "attention.cuh"
namespace ct {
bool attention_tc_supported(const AttentionArgs&) { return false; }
int attention_tc_forward(const AttentionArgs&, cudaStream_t) { return fail(CT_ERR_UNSUPPORTED, "attention_tc"); }
int64_t attention_tc_workspace(int64_t, int, int) { return 0; }
int attention_tc_backward(const AttentionArgs&, cudaStream_t) { return fail(CT_ERR_UNSUPPORTED, "attention_tc"); }
}  // namespace ct
