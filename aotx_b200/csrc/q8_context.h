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
    // The bytes that the latest mx4_quantize of this context wrote: a product whose weights they are waits for them
    // (other products may read their weights before the work before them has ended).
    const unsigned char *written[2];
    size_t written_bytes[2];
};
