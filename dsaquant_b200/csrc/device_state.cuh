// Per-device set-up shared by the library's entry points (defined in b200w4a4_api.cu).
#pragma once

namespace b200w4a4 {

struct DeviceInfo {
  int sm_count;
  int* status;           // time-out status word (a report)
  unsigned* abort_word;  // id of the launch that last timed out
};

// Capability check and one-time set-up of the current device; B200W4A4_OK or an error code.
__attribute__((visibility("hidden"))) int current_device(DeviceInfo* info);
// Id of a new launch on the current device (never 0), for a kernel that waits on barriers.
__attribute__((visibility("hidden"))) unsigned new_launch_id();
// cuTensorMapEncodeTiled, or null
__attribute__((visibility("hidden"))) void* tensor_map_encoder();

}  // namespace b200w4a4
