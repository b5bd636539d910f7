// What a launch of AdamW takes.
#pragma once
#include <hip/hip_runtime_api.h>
#include <stdint.h>

struct AdamWLaunch {
  const int64_t* shape;   // [ntensors][2]: elements, place in the arenas
  const void* chunks;     // [nchunks] {tensor, chunk of 2048 elements in it}
  void* live;             // [ntensors] written by the first kernel for the second: no two steps in flight may share it
  int* step;              // [ntensors]
  void* m;                // arenas: float, or e4m3 ...
  void* v;                // ... (r = sqrt(v) in 8 bits)
  float* m_scale;         // [arena / 256], 8 bits only
  float* r_scale;
  double lr, beta1, beta2;
  float b1, ob1, b2, ob2; // b, 1 - b, each rounded once
  float eps, decay;       // decay = 1 - lr * weight_decay
  float grad_scale;
  uint32_t seed;
  int ntensors, nchunks, bits;
};

// Bytes of `live` for each tensor.
extern "C" int dtf_sizeof_adamw_live();
// p, g, kind: host arrays of a->ntensors entries (g = 0: the tensor takes no part in this step; kind: bit 0 bf16 parameters, bit 1
// bf16 gradients)
extern "C" int dtf_adamw(const AdamWLaunch* a, const uint64_t* p, const uint64_t* g, const uint8_t* kind, hipStream_t st);
