// engine.hip - the translation unit of the expert engine: fronk_hip.hip and, behind
// it, what the dense operators (dense.h) ask of the engine. That stands here since
// counters of the engine's kernels (profiles/*_traffic.json) are bound to the bytes
// of fronk_hip.hip.
#include "fronk_hip.hip"

#include "dense.h"

namespace fronk {
int enter(void* stream, hipStream_t* out) {
  if (!g_open) return FR_HIP_STATE;
  CK(hipSetDevice(E.device));
  *out = !stream ? E.stream : stream == FR_HIP_STREAM_DEFAULT ? hipStream_t(nullptr) : static_cast<hipStream_t>(stream);
  return FR_HIP_OK;
}
}  // namespace fronk

extern "C" int fr_hip_device(void) { return g_open ? E.device : FR_HIP_STATE; }
