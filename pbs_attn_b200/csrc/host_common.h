// What the parts of the native host side share.
#pragma once

#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/object_ptr.h>

#include "../../include/pbs_b200.h"

inline bool capturing(cudaStream_t st) {
  cudaStreamCaptureStatus s;
  return cudaStreamIsCapturing(st, &s) != cudaSuccess || s != cudaStreamCaptureStatusNone;
}

// prefill.py's _readable
inline bool readable(const at::Tensor& t, bool distinct_heads) {
  const auto st = t.strides(), sz = t.sizes();
  if (st[3] != 1 || st[2] <= 0 || st[0] < 0 || st[1] < 0) return false;
  if (((st[0] | st[1] | st[2]) * t.element_size()) % 16 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  return !distinct_heads || ((st[0] > 0 || sz[0] == 1) && (st[1] > 0 || sz[1] == 1));
}

extern PyMethodDef pbs_decode_methods[];       // host_decode.cpp
