#include "gemm16.h"
using namespace tdh;
extern "C" {
size_t tdh_q8_row(int in) { return in > 0 ? (static_cast<size_t>(in) + 15) & ~static_cast<size_t>(15) : 0; }
}
