// What the library's translation units share on the host: the current device's state and the launch count (both live in
// nml_api.cu), and each file's kernels for the one-time set-up of a device.
#pragma once
#include <cuda.h>
#include <stdint.h>

#include <algorithm>

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

// Runs of `length` bytes, `step` apart (at least the length, where there are two).
struct Runs {
    uintptr_t at;
    long long count, length, step;
    uintptr_t end() const { return at + static_cast<uintptr_t>((count - 1) * step + length); }
};
// Whether a byte lies in both.
inline bool overlap(const Runs& x, const Runs& y) {
    if (x.end() <= y.at || y.end() <= x.at) return false;
    auto floor_div = [](long long v, long long by) { return v / by - (v % by < 0); };
    const Runs &a = x.count <= y.count ? x : y, &b = x.count <= y.count ? y : x;
    const long long from = static_cast<long long>(a.at - b.at);  // of a's first run, from b's
    if (a.count > 1 && a.step == b.step) {
        // run i of a begins `rest` into b's period ahead + i: it may reach b's run there, and the next one
        const long long ahead = floor_div(from, a.step), rest = from - ahead * a.step;
        auto meet = [&](long long shift) { return std::max(0ll, -shift) <= std::min(a.count - 1, b.count - 1 - shift); };
        return (rest < b.length && meet(ahead)) || (rest + a.length > a.step && meet(ahead + 1));
    }
    for (long long i = 0; i < a.count; ++i) {
        const long long first = from + i * a.step, step = b.count > 1 ? b.step : b.length;
        const long long lo = floor_div(first - b.length, step) + 1, hi = floor_div(first + a.length - 1, step);
        if (std::max(lo, 0ll) <= std::min(hi, b.count - 1)) return true;
    }
    return false;
}

// Loads a file's kernels and raises their shared-memory limits on the current device (called once per device).
NML_HIDDEN int prepare_logits_kernels();
NML_HIDDEN int prepare_ortho_kernels();

}  // namespace nml
