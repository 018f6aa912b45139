// Internal definitions of the adapter operators (include/laya_cuda_adapters.h).
#pragma once
#include "lc_common.cuh"

constexpr int kAdapterMaxRank = 256;

// Rows and adapters of one batch on the device (lc_adapter_plan_create).
struct AdapterPlan {
  int rows = 0, n_adapters = 0, nspans = 0;
  int32_t* dev = nullptr;          // one allocation behind the arrays below
  int32_t* row_adapter = nullptr;  // [rows]: the adapter of each row, -1 = none
  int2* spans = nullptr;           // [nspans]: row ranges, adapter by adapter, ascending within one
  int32_t* span_ptr = nullptr;     // [n_adapters + 1]: where each adapter's spans start
  cudaStream_t built_on = nullptr;
  cudaEvent_t built = nullptr;     // the arrays are on the device
  bool settled = false;            // `built` has been seen complete
  bool shared = false;             // used on another stream than built_on
};

void lc_adapters_destroy();
