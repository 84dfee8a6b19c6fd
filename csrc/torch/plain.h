// plain.h - what the native calls know for certain: plain CUDA tensors on the current device, no modes active, addresses.
#pragma once
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include "hccl/hccl_types.h"

namespace hcomm_torch {

static const c10::DispatchKeySet kPlain = c10::DispatchKeySet({c10::DispatchKey::Dense, c10::DispatchKey::AutogradFunctionality, c10::DispatchKey::ADInplaceOrView,
                                                        c10::DispatchKey::AutocastCUDA}) |
                                   c10::DispatchKeySet(c10::BackendComponent::CUDABit);

// A strided CUDA tensor with memory of its own on the current device, nothing wrapped around it; NULL otherwise.
inline const at::Tensor *Plain(PyObject *o, int device)
{
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.defined()) return nullptr;
    const c10::TensorImpl *impl = t.unsafeGetTensorImpl();
    if ((impl->key_set().raw_repr() & ~kPlain.raw_repr()) != 0 || !t.is_cuda() || t.get_device() != device || !impl->has_storage() || impl->layout() != c10::kStrided)
        return nullptr;
    return &t;
}
inline bool ModesActive()
{
    return at::impl::torch_function_mode_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set() ||
           (c10::impl::tls_local_dispatch_key_set().included_.raw_repr() & ~c10::default_included_set.raw_repr()) != 0;
}
// The device of this call, -1 where the general way has to be taken.
inline int Device() { return ModesActive() ? -1 : (int)c10::cuda::current_device(); }
inline void *StreamOf(int device) { return (void *)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }
// The address in a Python integer; false for anything else (the handle of a communicator that was destroyed is None).
inline bool Address(PyObject *o, void **p)
{
    if (!PyLong_Check(o)) return false;
    *p = PyLong_AsVoidPtr(o);
    if (!PyErr_Occurred()) return true;
    PyErr_Clear();
    return false;
}

inline int TypeCode(at::ScalarType t)
{
    switch (t) {
        case at::kChar: return HCCL_DATA_TYPE_INT8; case at::kShort: return HCCL_DATA_TYPE_INT16; case at::kInt: return HCCL_DATA_TYPE_INT32;
        case at::kLong: return HCCL_DATA_TYPE_INT64; case at::kByte: return HCCL_DATA_TYPE_UINT8; case at::kFloat: return HCCL_DATA_TYPE_FP32;
        case at::kHalf: return HCCL_DATA_TYPE_FP16; case at::kBFloat16: return HCCL_DATA_TYPE_BFP16; case at::kDouble: return HCCL_DATA_TYPE_FP64;
        default: return -1;
    }
}

}  // namespace hcomm_torch
