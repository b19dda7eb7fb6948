// Launch counter shared by all host wrappers (defined in gemm_tcgen05.cu).
#pragma once

namespace h3 {
void note_launch();
}  // namespace h3
