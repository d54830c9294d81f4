// A HIP runtime of 8 devices that runs nothing and writes down what it is asked for: loaded
// before libiekv_ops.so, its functions are the ones the library calls.
#include <cstddef>
#include <cstdint>
#include <cstdio>

namespace {
struct Dim3 {
  uint32_t x, y, z;
};
constexpr int kMost = 1 << 16;
struct Launch {
  int64_t device, grid_x, grid_y, block_x, stream;
} launches[kMost];
int n_launches = 0, current = 0, units_asked_of = -1, lds_asked_on = 0, devices = 8, last = 0;
Dim3 grid, block;
size_t shared;
void* stream;
}  // namespace

extern "C" {

int stub_launches() { return n_launches; }
void stub_forget() { n_launches = 0, units_asked_of = -1, lds_asked_on = 0; }
void stub_devices(int n) { devices = n; }
int stub_units_asked_of() { return units_asked_of; }
int stub_lds_asked_on() { return lds_asked_on; }   // a bit for each device
void stub_launch(int i, int64_t* out) {
  const Launch& l = launches[i];
  out[0] = l.device, out[1] = l.grid_x, out[2] = l.grid_y, out[3] = l.block_x, out[4] = l.stream;
}

int hipGetDevice(int* device) {
  *device = current;
  return 0;
}
int hipSetDevice(int device) {
  if (device < 0 || device >= devices) return last = 101;   // hipErrorInvalidDevice
  current = device;
  return 0;
}
int hipDeviceGetAttribute(int* value, int, int device) {
  units_asked_of = device;
  *value = 256 >> device;
  return 0;
}
int hipGetLastError() {
  const int error = last;
  last = 0;
  return error;
}
const char* hipGetErrorString(int error) { return error == 101 ? "invalid device" : "invalid launch"; }
int hipFuncSetAttribute(const void*, int, int) {
  lds_asked_on |= 1 << current;
  return 0;
}
int __hipPushCallConfiguration(Dim3 g, Dim3 b, size_t s, void* on) {
  grid = g, block = b, shared = s, stream = on;
  return 0;
}
int __hipPopCallConfiguration(Dim3* g, Dim3* b, size_t* s, void** on) {
  *g = grid, *b = block, *s = shared, *on = stream;
  return 0;
}
int hipLaunchKernel(const void*, Dim3 g, Dim3 b, void**, size_t, void* on) {
  // A dispatch counts its work-items in 32 bits.
  if (uint64_t(g.x) * b.x > UINT32_MAX || !g.x || !g.y || n_launches == kMost) return last = 9;
  launches[n_launches++] = {current, g.x, g.y, b.x, reinterpret_cast<int64_t>(on)};
  return 0;
}

}  // extern "C"
