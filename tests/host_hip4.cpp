// The stand-in HIP runtime of host_hip.cpp with what the 4-bit calls need beside it.
#include "host_hip.cpp"

extern "C" int hipFuncSetAttribute(const void *, int, int) { return kOk; }
