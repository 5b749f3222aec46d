// Host-side launchers of the paged-cache kernels.
#pragma once

#include <hip/hip_runtime.h>

#include "paged.hpp"

namespace nne {

hipError_t launch_paged_append(const PagedAppendParams& p, hipStream_t stream);
// p.cnt: B zeroed counters, left zeroed (not used without paths).
hipError_t launch_paged_commit(const PagedCommitParams& p, hipStream_t stream);
hipError_t launch_qk_norm_rope(const NormRopeParams& p, hipStream_t stream);
// One launch's sequences (p.b0, p.B <= kPagedSeqs), planned by paged_plan; p.ws
// holds the records that it asks for, of rec_rows rows, and p.cnt, where it asks
// for some, B * Hkv * n_rb zeroed counters, left zeroed.
hipError_t launch_paged_attention(const PagedAttnParams& p, hipStream_t stream);

}  // namespace nne
