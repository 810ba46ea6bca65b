// Span attention on fp16 (attention.h).
#include "attention.h"

int fa::attn::run_f16(const Params& p, hipStream_t s) { return launch_type<true>(p, s); }
