// Bindings that live outside hip_ext.cpp and join its module.
#pragma once

#include <pybind11/pybind11.h>

void register_core_ops(pybind11::module_& m);
