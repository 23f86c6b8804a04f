// Registers the language-model operators on the extension module.
#pragma once

#include <torch/extension.h>

namespace rl_amd {
void define_language_ops(py::module& m);
}
