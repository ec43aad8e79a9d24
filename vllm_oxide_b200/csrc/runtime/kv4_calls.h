// The calls of the 4-bit cache's operators (kv4_calls.cpp), as functions of the runtime module.
#pragma once
#include <Python.h>

namespace vob_calls {
PyMethodDef* methods();
}
