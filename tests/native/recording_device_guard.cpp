// Replaces PyTorch's CUDA device switch by one that only records, so that which device the
// binding makes current can be tested without a GPU.
#include <c10/core/impl/DeviceGuardImplInterface.h>

namespace {

int g_current = 0, g_log[64], g_count = 0;

struct Recorder final : c10::impl::DeviceGuardImplInterface {
  c10::DeviceType type() const override { return c10::kCUDA; }
  c10::Device exchangeDevice(c10::Device d) const override {
    const c10::Device old = getDevice();
    setDevice(d);
    return old;
  }
  c10::Device getDevice() const override { return {c10::kCUDA, static_cast<c10::DeviceIndex>(g_current)}; }
  void setDevice(c10::Device d) const override {
    g_current = d.index();
    if (g_count < 64) g_log[g_count++] = g_current;
  }
  void uncheckedSetDevice(c10::Device d) const noexcept override { setDevice(d); }
  c10::Stream getStream(c10::Device d) const override { return c10::Stream(c10::Stream::DEFAULT, d); }
  c10::Stream exchangeStream(c10::Stream s) const override { return s; }
  c10::DeviceIndex deviceCount() const noexcept override { return 4; }
};

}  // namespace

extern "C" void record_devices() {
  static const Recorder recorder;
  c10::impl::device_guard_impl_registry[static_cast<size_t>(c10::kCUDA)].store(&recorder);
}
extern "C" int recorded_devices(const int** at) {
  *at = g_log;
  return g_count;
}
