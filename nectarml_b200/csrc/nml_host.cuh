// What the library's translation units share on the host: the current device's state and the launch count (both live in
// nml_api.cu), and each file's kernels for the one-time set-up of a device.
#pragma once
#include <cuda.h>
#include <stdint.h>

#define NML_HIDDEN __attribute__((visibility("hidden")))

namespace nml {

// The word where kernels of the current device report an abandoned wait, and how many SMs a launch may occupy.  Sets the
// device up on its first call (see nml_init).  Returns a status.
NML_HIDDEN int current_device(int** status_word, int* sms);
NML_HIDDEN int usable_sms();  // the same count without touching a device: for plans made where there may be none
NML_HIDDEN void count_launches(int n);
// Keeps the text of a CUDA error for nml_status_string; returns NML_ERR_CUDA.
NML_HIDDEN int cuda_failed(int error, const char* what);

// Tensor map of a dense tensor of fp16 elements, fastest dimension first, unswizzled.  Returns a status.
NML_HIDDEN int encode_box(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint32_t* box);

// Loads a file's kernels and raises their shared-memory limits on the current device (called once per device).
NML_HIDDEN int prepare_logits_kernels();
NML_HIDDEN int prepare_ortho_kernels();

}  // namespace nml
