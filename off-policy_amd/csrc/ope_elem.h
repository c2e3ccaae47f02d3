// Element types of the memory-block operators (ope_delta*.hip, ope_norm.hip, ope_linear.hip): float32, bfloat16, float16 in memory, float32
// in every register. Conversions are the compiler's: widening is exact, narrowing rounds to nearest even.
#pragma once
#include "ope_common.h"

namespace ope {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef float f32x8 __attribute__((ext_vector_type(8)));

// N elements that lie behind each other, aligned to ONE element only: gfx950 takes wide loads at any element address, and the type tells the
// compiler not to assume more. Rows of odd width need no scalar path this way.
template <typename T, int N>
struct Pack {
  typedef T vec __attribute__((ext_vector_type(N)));
  typedef vec loose __attribute__((aligned(sizeof(T))));
  typedef float fvec __attribute__((ext_vector_type(N)));
};
template <typename T, int N>
__device__ __forceinline__ typename Pack<T, N>::fvec load_pack(const T* p) {
  typename Pack<T, N>::vec v = *reinterpret_cast<const typename Pack<T, N>::loose*>(p);
  return __builtin_convertvector(v, typename Pack<T, N>::fvec);
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, typename Pack<T, N>::fvec f) {
  *reinterpret_cast<typename Pack<T, N>::loose*>(p) = __builtin_convertvector(f, typename Pack<T, N>::vec);
}

// A launch holds fewer than 2^32 threads; what would pass that is refused with the arguments, not left to the runtime.
static inline bool launch_fits(int64_t blocks, int threads) { return blocks < ((int64_t)1 << 32) / threads; }

static inline int elem_bytes(int dtype) { return dtype == OPE_F32 ? 4 : (dtype == OPE_E4M3 ? 1 : 2); }
static inline bool elem_float(int dtype) { return dtype == OPE_F32 || dtype == OPE_BF16 || dtype == OPE_F16; }

// f(T{}) for the type that `dtype` names
template <typename F>
static inline int with_elem(int dtype, F f) {
  switch (dtype) {
    case OPE_F32: return f(float{});
    case OPE_BF16: return f(bf16_t{});
    case OPE_F16: return f(f16_t{});
  }
  return OPE_EINVAL;
}

}  // namespace ope
