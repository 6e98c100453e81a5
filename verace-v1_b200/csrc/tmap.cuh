// Host side of the TMA tensor maps: the driver's cuTensorMapEncodeTiled, resolved once
// through the runtime (the library links no driver import library).
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

namespace verace {

// The entry point (with a context bound first, on a thread that has none); nullptr when the driver does not provide it.
PFN_cuTensorMapEncodeTiled_v12000 tmap_encoder();

}  // namespace verace
