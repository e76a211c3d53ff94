// The handle of the PagedAttention operator, shared by the files that implement its entry points (pa_api.cu, masked_api.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <string>
#include <vector>

#include "../../include/masked_b200.h"
#include "pa_kernels.h"

struct pa_handle {
    pa_model_desc desc;
    pa::CacheGeom g;
    int device = 0;
    int sm_count = 148;
    cudaStream_t stream = nullptr;
    uint8_t* ws = nullptr;       // kernel scratch
    size_t ws_bytes = 0;
    uint32_t* status = nullptr;  // device status word
    uint8_t* stage_dev = nullptr;  // device copies of host tensors (forward_host)
    size_t stage_dev_bytes = 0;
    uint8_t* stage_host = nullptr;  // pinned
    size_t stage_host_bytes = 0;
    int64_t launches = 0;
    int last_prefill_kernel = PA_PREFILL_NONE;
    bool force_generic_prefill = false;        // env PA_B200_GENERIC_PREFILL=1: cross-check path
    bool test_drop_copy = false;               // env PA_B200_TEST_DROP_FIRST_COPY=1: the decode kernel's bounded wait is made to run out
    bool timing = false;                       // record events around the split-K decode kernel
    std::vector<cudaEvent_t> ev;               // pairs, created on demand
    size_t ev_used = 0;
    // masked steps (masked_api.cu)
    uint8_t* mws = nullptr;       // their scratch
    size_t mws_bytes = 0;
    bool mws_captured = false;    // a stream capture has named it
    std::vector<uint8_t*> mws_retired;   // scratch of captures, outgrown since: their graphs may still run
};

namespace pa {
void set_last_error(const std::string& msg);

// pa_api.cu
int validate_forward_args(const pa_handle* h, const pa_forward_args* a);
// The host-tensor entry points; `mask` null: a causal step.
int forward_host(pa_handle* h, const pa_forward_args* a, const pa_mask_args* mask);

// masked_api.cu: a masked step of device tensors whose arguments have been checked.
int forward_masked(pa_handle* h, const pa_forward_args* a, const pa_mask_args& mask, cudaStream_t stream);
}  // namespace pa
