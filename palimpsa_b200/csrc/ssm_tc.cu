#include "ssm.cuh"
namespace palimpsa {
bool ssm_tc_supported(const palimpsa_ssm&) { return false; }
size_t ssm_tc_state_bytes(const palimpsa_ssm&, long long, bool) { return 0; }
size_t ssm_tc_workspace_bytes(const palimpsa_ssm&, long long) { return 0; }
int ssm_tc_fwd(const SsmArgs&, bool, cudaStream_t) { return PALIMPSA_E_LAUNCH; }
int ssm_tc_bwd(const SsmArgs&, cudaStream_t) { return PALIMPSA_E_LAUNCH; }
}  // namespace palimpsa
