// The feed-forward operators' part of the Python module.
#pragma once

#include <torch/extension.h>

void register_projection_ops(py::module& m);
