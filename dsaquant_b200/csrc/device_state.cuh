// Per-device set-up shared by the library's entry points (defined in b200w4a4_api.cu).
#pragma once

namespace b200w4a4 {

// Capability check and one-time set-up of the current device; B200W4A4_OK or an error code.
// sm_count / status: its SM count and the address of its time-out status word.
__attribute__((visibility("hidden"))) int current_device(int* sm_count, int** status);

}  // namespace b200w4a4
