// The attention kernels of a bf16 cache (a file to each type: they build side by side).
#include "attention_kernels.hpp"

namespace sarek_hip {
int launch_attention_bf16(const AttentionArgs &s, const Launch &own, const Launch *before, hipStream_t st) { return launch_type<Bf16>(s, own, before, st); }
}  // namespace sarek_hip
