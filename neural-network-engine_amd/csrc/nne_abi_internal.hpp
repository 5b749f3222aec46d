// Pieces of the C ABI (abi.cpp) that other sources of the library share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "nne_attn.h"

namespace nne {

// Sets the calling thread's nne_last_error() message and returns `code`.
int fail_message(int code, const char* msg);
int fail_hip(hipError_t e, const char* what);

// Body of nne_decode_attention / nne_decode_step (k_new == NULL: attention
// only).  Validates every argument, then launches.  A NULL workspace makes
// the call use the stream's library-side one.
int run_decode(const float* q, const int64_t* q_strides, const float* k_cache, const float* v_cache,
               const int32_t* lens_dev, int32_t* lens_dev_w, int32_t* lens_host, const float* k_new,
               const int64_t* kn_strides, const float* v_new, const int64_t* vn_strides, float* o,
               const int64_t* o_strides, int64_t B, int64_t Hq, int64_t Hkv, int64_t capacity,
               int64_t d, int has_scale, float scale, const nne_workspace_t* ws, hipStream_t s);

// nne_last_error() message in printf form; returns `code`.
int fail_format(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// Row-major strides of a [n0, n1, n2, n3] tensor.
void row_major_strides(const int64_t* shape, int64_t* strides);

// CUs of the current device.
int cus_of_device();

// Records and counters of one call: the caller's workspace, checked against the
// call's needs, or (ws == NULL) the stream's library-side ones.  A stream under
// capture is refused one that would have to be allocated: the allocation would
// become a node of the graph.
int take_workspace(const nne_workspace_t* ws, uint64_t need_bytes, int64_t need_counters,
                   hipStream_t s, void** records, uint32_t** counters, const char* what);

}  // namespace nne
