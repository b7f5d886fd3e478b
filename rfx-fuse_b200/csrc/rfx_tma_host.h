// The driver's tensor-map encoder (rfx_lowrank_host.cu), shared by the tensor-core hosts.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

namespace rfxh {
PFN_cuTensorMapEncodeTiled_v12000 encode_fn();  // throws RfxError when the driver has none
}  // namespace rfxh
