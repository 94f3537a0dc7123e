// What the adapters of the torch.ops.npu.* operators share: status and device checks, the current stream, allocation.
#pragma once
#include <ATen/ATen.h>
#include <ATen/DimVector.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <mutex>

#include "mi355_quant.h"

namespace mi355_ops {
// A stream's workspace, its zero area (MI355_WORKSPACE_ZERO_BYTES) zero (npu_ops.cpp).  It is this call's as long as the object
// lives: keep it until the last launch that uses it is enqueued, and take no second one meanwhile.
struct Workspace {
    std::unique_lock<std::mutex> held;
    at::Tensor memory;
};
Workspace workspace(const at::Tensor &like, size_t bytes, bool large_for_call = false);
} // namespace mi355_ops

namespace {

using at::Tensor;
using c10::optional;
using mi355_ops::Workspace;

void check_status(int status, const char *op)
{
    TORCH_CHECK(status == MI355_OK, op, ": ", mi355_status_string(status), " (status ", status, ")");
}

// Same text as the reference's generated wrapper check (asserted by
// test/custom_ops/test_npu_anti_quant.py:86-88).
void check_same_device(const char *op, std::initializer_list<const Tensor *> ts)
{
    const Tensor *first = nullptr;
    for (const Tensor *t : ts) {
        if (!t || !t->defined()) continue;
        if (!first) {
            first = t;
            continue;
        }
        TORCH_CHECK(t->device() == first->device(),
                    "Expected all tensors to be on the same device, but found at least two devices, ", first->device(),
                    " and ", t->device(), "! (when checking arguments for ", op, ")");
    }
}

const Tensor *opt(const optional<Tensor> &t) { return t.has_value() && t->defined() ? &*t : nullptr; }

void *stream_of(const Tensor &t)
{
    // PyTorch-ROCm names its HIP device type "cuda"; these are its stream/guard classes for that device type
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// An uninitialised contiguous tensor beside `like`: through the dispatcher for shape inference (kMeta), and straight from the
// caching allocator for a launch (kLaunch), where the dispatcher and the option parsing would be a tenth of an operator's host
// time at decode sizes for each output.
enum Alloc { kMeta, kLaunch };
Tensor new_empty(Alloc how, const Tensor &like, at::IntArrayRef sizes, at::ScalarType dtype)
{
    if (how == kLaunch) return Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt));
    return at::empty(sizes, like.options().dtype(dtype));
}

// (at::contiguous dispatches even when there is nothing to do)
Tensor packed(const Tensor &t) { return t.is_contiguous() ? t : t.contiguous(); }

} // namespace
