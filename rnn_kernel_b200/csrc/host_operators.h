// host_operators.cpp's part of the Python module rnn_kernel_b200._host.
#pragma once

#include <Python.h>

PyMethodDef* operator_methods();
