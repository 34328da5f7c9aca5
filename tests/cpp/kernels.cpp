// Names of the kernels that a library registers, and of those that it has launched since they were
// last asked for. Loaded before launches.cpp's stand-in for HIP, which has the other calls.
#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <map>
#include <set>
#include <string>

namespace {
std::map<const void*, std::string>& registered() {
  static std::map<const void*, std::string> names;
  return names;
}
std::set<std::string> g_launched;
std::string g_text;

template <class Names, class F>
const char* lines(const Names& names, F name) {
  g_text.clear();
  for (const auto& n : names) g_text += name(n) + "\n";
  return g_text.c_str();
}
}  // namespace

extern "C" {

const char* kernels_registered() {
  return lines(registered(), [](const auto& n) { return n.second; });
}
const char* kernels_launched() {
  lines(g_launched, [](const auto& n) { return n; });
  g_launched.clear();
  return g_text.c_str();
}

void** __hipRegisterFatBinary(const void*) {
  static void* modules = nullptr;
  return &modules;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, dim3*, dim3*, int*) {
  registered()[host] = name;
}
void __hipRegisterVar(void**, void*, char*, char*, int, std::size_t, int, int) {}
hipError_t hipLaunchKernel(const void* kernel, dim3, dim3, void**, std::size_t, hipStream_t) {
  g_launched.insert(registered()[kernel]);
  return hipSuccess;
}

}  // extern "C"
