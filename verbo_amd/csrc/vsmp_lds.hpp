// A kernel's dynamic LDS limit (host code).
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <initializer_list>
#include <mutex>

namespace vsmp {

// Raises the dynamic LDS limit of kernels above the default, once per device: the attribute
// belongs to each device's instance of a kernel, so a process that launches on several devices
// sets it on each (devices 64 and up are set at every launch).
struct DynLdsOnce {
  std::atomic<unsigned long long> done{0};
  std::mutex m;
};
inline void allow_dyn_lds(DynLdsOnce& o, std::initializer_list<const void*> fns, int bytes) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return;
  const unsigned long long bit = (dev >= 0 && dev < 64) ? 1ull << dev : 0ull;
  if (bit && (o.done.load(std::memory_order_acquire) & bit)) return;
  std::lock_guard<std::mutex> g(o.m);
  if (bit && (o.done.load(std::memory_order_relaxed) & bit)) return;
  for (const void* fn : fns) (void)hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  o.done.fetch_or(bit, std::memory_order_release);
}

}  // namespace vsmp
