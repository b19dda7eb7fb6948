// The bounds-checked build of attn/packed_fwd.cu (module h3_a100._C_checked).
#include "../attn/packed_fwd.cu"
