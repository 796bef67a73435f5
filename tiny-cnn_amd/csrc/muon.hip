#include "gemm16.h"
using namespace tdh;
extern "C" {
void tdh_muon_default(tdh_muon *o) {
  if (!o) return;
  *o = tdh_muon{0.02f, 0.95f, 0.0f, 1.0f, 1, 5, 3.4445f, -4.7750f, 2.0315f, 1e-7f, TDH_F32};
}
}
