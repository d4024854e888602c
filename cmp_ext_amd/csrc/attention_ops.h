// The attention operators' part of the Python module.
#pragma once

#include <torch/extension.h>

void register_attention_ops(py::module& m);
