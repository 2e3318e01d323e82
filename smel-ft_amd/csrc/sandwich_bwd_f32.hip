#include "sandwich_bwd.h"

int smel::sandwich_bwd_f32(SwArgs& a, hipStream_t stream) { return sandwich_bwd_rows<2>(a, stream); }
