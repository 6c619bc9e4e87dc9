// The training-step operators' part of the extension module.
#pragma once

#include <torch/extension.h>

void bind_training(py::module& m);
