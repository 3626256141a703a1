#pragma once
#include <Python.h>

// The operators of train/capi_train.h on tensors; they end with an empty entry.
PyMethodDef *train_methods();
