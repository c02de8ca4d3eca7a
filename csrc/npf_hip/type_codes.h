// Codes that the bindings pass to the kernels for a tensor's type.
#pragma once

enum NpfType { NPF_F32 = 0, NPF_BF16 = 1, NPF_F16 = 2, NPF_F64 = 3 };
