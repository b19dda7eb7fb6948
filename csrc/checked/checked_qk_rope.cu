// The bounds-checked build of rope/qk_rope.cu (module h3_a100._C_checked).
#include "../rope/qk_rope.cu"
