#include "sandwich_bwd.h"

int smel::sandwich_bwd_f16(SwArgs& a, hipStream_t stream) { return sandwich_bwd_rows<1>(a, stream); }
