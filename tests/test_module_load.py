"""What nc_module_load_embedded loads, and when: hip_api.cpp against a HIP runtime of counters, on the CPU."""

import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "not-cute-zig_amd", "csrc")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

STUB = r'''
#include <hip/hip_runtime_api.h>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include "notcute_flash.h"

extern "C" {
int nc_internal_noalloc_setup(void) { return 0; }
int nc_internal_module_kept_function(nc_module, uint32_t, const char *, nc_function *);
}

// the embedded objects, of one byte each
asm(R"(
    .pushsection .rodata
    .globl nc_embedded_code_object, nc_embedded_code_object_end, nc_embedded_paged_object
nc_embedded_code_object: .byte 1
nc_embedded_code_object_end:
nc_embedded_paged_object: .byte 2
    .popsection
)");

int device = 0, flash_loads = 0, paged_loads = 0, paged_unloads = 0, paged_device = -1, broken = 0;
hipStreamCaptureMode mode = hipStreamCaptureModeGlobal, paged_mode = hipStreamCaptureModeGlobal;
char flash_object, paged_object;

extern "C" {
hipError_t hipGetDevice(int *d) { *d = device; return hipSuccess; }
hipError_t hipSetDevice(int d) { device = d; return hipSuccess; }
const char *hipGetErrorName(hipError_t) { return "error"; }
hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode *m) {
    const hipStreamCaptureMode was = mode;
    mode = *m;
    *m = was;
    return hipSuccess;
}
hipError_t hipModuleLoadData(hipModule_t *m, const void *image) {
    if (*(const unsigned char *)image == 1) {
        ++flash_loads;
        *m = (hipModule_t)&flash_object;
        return hipSuccess;
    }
    if (broken) return hipErrorOutOfMemory;
    ++paged_loads;
    paged_device = device;
    paged_mode = mode;
    *m = (hipModule_t)&paged_object;
    return hipSuccess;
}
hipError_t hipModuleUnload(hipModule_t m) { paged_unloads += m == (hipModule_t)&paged_object; return hipSuccess; }
hipError_t hipModuleGetFunction(hipFunction_t *f, hipModule_t m, const char *name) {
    const bool paged = std::strncmp(name, "nc_paged_", 9) == 0;
    if (m != (hipModule_t)(paged ? &paged_object : &flash_object)) return hipErrorNotFound;
    *f = (hipFunction_t)name;
    return hipSuccess;
}
}

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    nc_module a = nullptr, b = nullptr;
    nc_function f = nullptr, g = nullptr;
    // a program that only uses the flash forward
    CHECK(nc_module_load_embedded(&a) == NC_SUCCESS && nc_module_get_function(&f, a, "nc_flash") == NC_SUCCESS);
    CHECK(flash_loads == 1 && paged_loads == 0);
    CHECK(nc_module_unload(a) == NC_SUCCESS && paged_unloads == 0);
    // the cache's kernels: once, on the module's device whatever the current one, and under a capture
    CHECK(nc_module_load_embedded(&a) == NC_SUCCESS);
    device = 3;
    CHECK(nc_internal_module_kept_function(a, 0, "nc_paged_build", &f) == NC_SUCCESS && f);
    CHECK(nc_internal_module_kept_function(a, 0, "nc_paged_build", &g) == NC_SUCCESS && g == f);
    CHECK(nc_module_get_function(&g, a, "nc_paged_append_rows") == NC_SUCCESS);
    CHECK(paged_loads == 1 && paged_device == 0 && device == 3);
    CHECK(paged_mode == hipStreamCaptureModeRelaxed && mode == hipStreamCaptureModeGlobal);
    device = 0;
    // where they cannot be loaded the flash forward can still be used, and they are tried again
    broken = 1;
    CHECK(nc_module_load_embedded(&b) == NC_SUCCESS && nc_module_get_function(&f, b, "nc_flash") == NC_SUCCESS);
    CHECK(nc_internal_module_kept_function(b, 0, "nc_paged_build", &f) == NC_ERROR_OUT_OF_MEMORY);
    CHECK(nc_module_get_function(&f, b, "nc_flash_other") == NC_SUCCESS);
    broken = 0;
    CHECK(nc_internal_module_kept_function(b, 0, "nc_paged_build", &f) == NC_SUCCESS && paged_loads == 2);
    CHECK(nc_module_unload(a) == NC_SUCCESS && nc_module_unload(b) == NC_SUCCESS && paged_unloads == 2);
    // a module loaded from data has no such kernels
    const unsigned char image[] = {1};
    CHECK(nc_module_load_data(&a, image) == NC_SUCCESS);
    CHECK(nc_internal_module_kept_function(a, 0, "nc_paged_build", &f) == NC_ERROR_NOT_FOUND && paged_loads == 2);
    CHECK(nc_module_unload(a) == NC_SUCCESS);
    return 0;
}
'''


def test_cache_kernels_are_loaded_when_first_asked_for(tmp_path):
    src, exe = tmp_path / "load.cpp", tmp_path / "load"
    src.write_text(STUB)
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"), "-I", CSRC, "-I",
                    os.path.join(ROCM, "include"), str(src), os.path.join(CSRC, "hip_api.cpp"), "-o", str(exe),
                    "-Wl,--unresolved-symbols=ignore-all"], check=True, capture_output=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr
