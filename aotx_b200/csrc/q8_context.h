// The per-device context behind both C interfaces (include/aotx_q8_b200.h, include/aotx_mx4_b200.h).
#pragma once

#include "q8_launch.h"

struct aotx_q8_ctx {
    int device;
    unsigned int sm_count;
    int path;
    int last_cuda;
    int overlap;
    unsigned int launches;
    q8::UmmaScratch scratch;
};
