// What the translation units of the CPython module kernel._bind share: tensors
// as descriptors of the C-ABI, statuses as exceptions, and the checks that every
// differentiable operator makes before it builds its autograd node.
#pragma once
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>

#include "saf_attn.h"

namespace saf_bind {

// dtype code of the C-ABI, -1 for a dtype that is no activation's, weight's or index's
int dtype_code(at::ScalarType t);

// A dual tensor: none of the operators has a forward-mode derivative, and
// their results would drop the tangent without a word.
bool has_tangent(const at::Tensor& x);

// The exception of a status, with the library's message.
void check(int rc);

// saf_tensor_t of a tensor; an undefined one is absent, one of more dimensions than
// a descriptor has is refused.
saf_tensor_t desc(const char* what, const at::Tensor& x);

// A leaf's autograd node belongs to the stream of the call that made it.  A
// captured backward would make that stream wait for the capturing one, and with
// it join the capture without ever leaving it: torch ends the process there.
// So tensors that are such a leaf, or come from one by operations of a single
// input (views, slices, casts), are refused.
void refuse_foreign_capture(const char* what, const char* name, const at::Tensor& x);

// The gradient as it is, or, where the backward pass itself is recorded, one
// whose derivative is refused.
at::Tensor only_once(const char* what, at::Tensor dx);

// The tensor as a new Python object; None for an undefined one.
PyObject* wrap(const at::Tensor& t);

// py_bind_train.cpp
PyObject* embed_tokens(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* add_layernorm(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* gelu_packed(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* gelu_packed_bwd(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* pack_activation(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* unpack_activation(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* check_differentiable(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* library_train(PyObject*, PyObject* const* args, Py_ssize_t n);

}  // namespace saf_bind
