// Single translation unit of libwanflash: the device error word and wait
// limit are shared by every kernel, so the library is compiled as one unit
// (no relocatable device code or device link step needed).
#include "wf_capi.cu"
#include "wf_fwd.cu"
#include "wf_fwd2.cu"
#include "wf_bwd.cu"
#include "wf_bwd2.cu"
#include "wf_aux.cu"
#include "wf_noalloc.cu"
#include "wf_rope.cu"
#include "wf_decode.cu"
#include "wf_packed_plan.cu"
#include "wf_packed_fwd.cu"
#include "wf_packed_bwd.cu"
#include "wf_packed_capi.cu"
