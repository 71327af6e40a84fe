// Element types of the row lookup and the gated recurrence: what is held in memory (bf16, fp16, fp32, fp64) and the
// type their sums and states are kept in (fp32; fp64 for fp64).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>
#include <stdexcept>

namespace lga {

enum SeqType : int64_t { kBf16 = 0, kF16 = 1, kF32 = 2, kF64 = 3 };

template <typename T> struct WideOf { typedef float type; };
template <> struct WideOf<double> { typedef double type; };
template <typename T> using Wide = typename WideOf<T>::type;

__device__ __forceinline__ float fma_wide(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_wide(double a, double b, double c) { return __builtin_fma(a, b, c); }

// V neighbouring elements, loaded and stored as words of up to 16 bytes wherever they start: global memory takes them at
// any multiple of the element's size.  Where V does not divide a row, the row's last pack starts V before its end and
// shares elements with the one before; both hold the same values of them.
template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[V]; };

template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}
template <typename T, int V> __device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& x) {
  *reinterpret_cast<Pack<T, V>*>(p) = x;
}

// Makes the tensors' device current for the launch and puts the caller's back.
class DeviceScope {
 public:
  explicit DeviceScope(int64_t device) {
    if (hipGetDevice(&before_) != hipSuccess) throw std::runtime_error("no current HIP device");
    if ((int64_t)before_ != device) {
      if (hipSetDevice((int)device) != hipSuccess) throw std::runtime_error("cannot select the tensors' device");
      changed_ = true;
    }
  }
  ~DeviceScope() { if (changed_) (void)hipSetDevice(before_); }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;

 private:
  int before_ = 0;
  bool changed_ = false;
};

}  // namespace lga
