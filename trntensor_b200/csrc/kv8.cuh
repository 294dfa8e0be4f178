// Paged key-value cache held in 8 bits: storage order and shared helpers.
//
// A page holds P tokens (16, 32, 64 or 128) of every kv head; keys and values
// have one fp32 scale for each page and head, x^ = s c with c in -127..127.
// Codes are stored biased by 128 (a byte above 0x6400 or below 0x64 then is the
// fp16 number 1024 + c + 128). A page and head is P / 16 units of 16 tokens:
//   keys    [page][head][unit][token 16][D]
//   values  [page][head][unit][D][token 16]
// so that the tensor-core fragments of both products read 16 neighbouring
// bytes a lane, and a unit of either is 16 D neighbouring bytes, which a bulk
// copy takes at once.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace tt {
namespace kv8 {

// Bits of a cache's status word, set by the kernels and read by the caller.
enum Status : int {
  kBadPage = 1,    // a page id outside the cache (its tokens are left out)
  kBadLength = 2,  // a length or count that is negative or passes the table
  kSharedPage = 4, // one call writes a page for two places
  kTimeout = 8     // a copy never arrived
};

__device__ __forceinline__ void raise(int* status, int bit) { atomicOr(status, bit); }

// Angle of position t and frequency f (32 bits), exact to fp32 for any t: the
// product and the reduction to one turn are made in 64 bits.
__device__ __forceinline__ void turn(long long t, float f, float* c, float* s) {
  const double a = (double)t * (double)f;
  const double r = a - rint(a * 0.15915494309189535) * 6.283185307179586;
  sincosf((float)r, s, c);
}

}  // namespace kv8
}  // namespace tt
