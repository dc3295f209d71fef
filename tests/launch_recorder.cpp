// Stands in for the HIP runtime in a process without a GPU: kernels of a library that is loaded after this one are
// noted by name when they are registered, and with their grid when they are launched.  None runs.
#include <cstddef>
#include <cstdint>
#include <map>
#include <string>

namespace {
struct Dim3 {
    uint32_t x, y, z;
};
std::map<const void *, std::string> names;
std::string launched, answer;
Dim3 grid, block;
size_t shared;
void *on;
}  // namespace

extern "C" {
void **__hipRegisterFatBinary(const void *) {
    static void *module;
    return &module;
}
void __hipUnregisterFatBinary(void **) {}
void __hipRegisterVar(void **, void *, char *, const char *, int, size_t, int, int) {}
void __hipRegisterFunction(void **, const void *host, char *, const char *name, unsigned, void *, void *, void *, void *, int *) { names[host] = name; }

int __hipPushCallConfiguration(Dim3 g, Dim3 b, size_t bytes, void *stream) {
    grid = g, block = b, shared = bytes, on = stream;
    return 0;
}
int __hipPopCallConfiguration(Dim3 *g, Dim3 *b, size_t *bytes, void **stream) {
    *g = grid, *b = block, *bytes = shared, *stream = on;
    return 0;
}
int hipLaunchKernel(const void *host, Dim3 g, Dim3 b, void **, size_t, void *) {
    launched += names[host];
    for (uint32_t n : {g.x, g.y, g.z, b.x, b.y, b.z}) launched += ' ' + std::to_string(n);
    launched += '\n';
    return 0;
}
int hipGetLastError() { return 0; }

// "name grid.x grid.y grid.z block.x block.y block.z" of every launch since the last call
const char *recorded_launches() {
    answer = launched;
    launched.clear();
    return answer.c_str();
}
const char *registered_kernels() {
    answer.clear();
    for (const auto &kernel : names) answer += kernel.second + '\n';
    return answer.c_str();
}
}
