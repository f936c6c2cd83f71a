// Operators of a transformer block on token tensors (attention, layer norm, rotary positions): registered into _C.
#pragma once
#include <torch/extension.h>

void bind_block_ops(py::module_& m);
