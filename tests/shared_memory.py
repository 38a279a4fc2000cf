"""A kernel that leaves a value in the shared memory of every SM, to put ahead of one whose results must not depend on what
it finds there."""
import functools

import torch
from cuda.bindings import driver, nvrtc

# One block takes an SM to itself; it stays for 50 us, so that a block per SM is on each of them. `seen`: the SMs' numbers.
SOURCE = rb"""
extern "C" __global__ void fill(unsigned value, int words, unsigned* seen) {
  extern __shared__ volatile unsigned memory[];
  for (int i = threadIdx.x; i < words; i += blockDim.x) memory[i] = value;
  if (threadIdx.x == 0) {
    unsigned sm;
    asm volatile("mov.u32 %0, %%smid;" : "=r"(sm));
    seen[blockIdx.x] = sm;
    for (int i = 0; i < 50; ++i) __nanosleep(1000);
  }
}
"""


def _ok(result):
    assert int(result[0]) == 0, result[0]
    return result[1] if len(result) > 1 else None


@functools.cache
def _kernel():
    torch.cuda.current_stream().synchronize()   # makes the context current
    program = _ok(nvrtc.nvrtcCreateProgram(SOURCE, b"fill.cu", 0, [], []))
    _ok(nvrtc.nvrtcCompileProgram(program, 1, [b"--gpu-architecture=sm_100a"]))
    image = b" " * _ok(nvrtc.nvrtcGetCUBINSize(program))
    _ok(nvrtc.nvrtcGetCUBIN(program, image))
    kernel = _ok(driver.cuModuleGetFunction(_ok(driver.cuModuleLoadData(image)), b"fill"))
    most = torch.cuda.get_device_properties(0).shared_memory_per_block_optin
    _ok(driver.cuFuncSetAttribute(kernel, driver.CUfunction_attribute.CU_FUNC_ATTRIBUTE_MAX_DYNAMIC_SHARED_SIZE_BYTES, most))
    return kernel, most


def fill(bits):
    """Every 32-bit word of what a block may have becomes `bits`, on all SMs. Returns the SMs' numbers (on the device)."""
    import ctypes
    kernel, most = _kernel()
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    seen = torch.empty(sms, dtype=torch.int32, device="cuda")
    args = ((bits, most // 4, seen.data_ptr()), (ctypes.c_uint, ctypes.c_int, ctypes.c_void_p))
    _ok(driver.cuLaunchKernel(kernel, sms, 1, 1, 1024, 1, 1, most, torch.cuda.current_stream().cuda_stream, args, 0))
    return seen
