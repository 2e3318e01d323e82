#include "sandwich_bwd.h"

int smel::sandwich_bwd_bf16(SwArgs& a, hipStream_t stream) { return sandwich_bwd_rows<0>(a, stream); }
