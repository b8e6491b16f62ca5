// Registers the operators of a decoder's training step with the Python module.
#pragma once
#include <pybind11/pybind11.h>

void register_decoder(pybind11::module_& m);
