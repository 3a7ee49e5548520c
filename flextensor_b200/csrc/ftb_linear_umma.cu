#include "ftb_linear.h"
namespace ftb {
int launch_linear_umma(const LinArgs&, const ftb_config*, int*, cudaStream_t) { return FTB_E_UNSUPPORTED; }
}
