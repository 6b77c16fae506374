// What a linear's epilogue does with a sum y (fp32): act(y + bias) + residual, rounded once to the output's type.
#pragma once
#include "common.h"

namespace ifd {

enum EpiAct { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4 };

struct Epi {
  const uint16_t* bias = nullptr;  // bf16 [N], or null
  const uint16_t* res = nullptr;   // bf16 [M][ldr], or null; may be C itself
  int ldr = 0;
  int act = kActNone;
};

__device__ __forceinline__ float epi_act(float v, int act) {
  switch (act) {  // uniform over the launch
    case kActRelu: return v < 0.f ? 0.f : v;
    case kActSilu: return v / (1.f + expf(-v));
    case kActGelu: return v * 0.5f * erfcf(v * -0.70710678118654752f);
    case kActGeluTanh: return v / (1.f + expf(-1.5957691216057308f * (v + 0.044715f * v * v * v)));
    default: return v;
  }
}

}  // namespace ifd
