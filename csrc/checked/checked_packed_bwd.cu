// The bounds-checked build of attn/packed_bwd.cu (module h3_a100._C_checked).
#include "../attn/packed_bwd.cu"
