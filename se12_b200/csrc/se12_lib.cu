// Single translation unit of libse12_b200.so: the kernels share the device
// status word g_status, so they are compiled together.
#include "se12_codec.cu"
#include "se12_gemv.cu"
#include "se12_chain.cu"
#include "se12_abi.cu"
#include "se12_kv.cu"
#include "se12_kv4.cu"
#include "se12_attend.cu"
#include "se12_attend4.cu"
#include "se12_attend_tile.cu"
#include "se12_logprobs.cu"
#include "se12_serve_abi.cu"
