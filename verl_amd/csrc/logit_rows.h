// Rows of materialised logits, shared by the kernels that walk them: element types, 16-byte groups, dispatch.
#pragma once
#include <type_traits>

#include "common.h"

namespace vamd {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegBig = -1.0e30f;
constexpr int kInFlight = 4;  // 16-byte loads a thread issues before it consumes them

// kVec: elements per 16-byte load; kBackwardLoads: such loads per thread in the backward kernel
struct F32 { using type = float; static constexpr int kVec = 4; static constexpr int kBackwardLoads = 2; };
struct BF16 { using type = uint16_t; static constexpr int kVec = 8; static constexpr int kBackwardLoads = 1; };
struct F16 { using type = _Float16; static constexpr int kVec = 8; static constexpr int kBackwardLoads = 1; };

__device__ __forceinline__ float to_float(float x, F32) { return x; }
__device__ __forceinline__ float to_float(uint16_t x, BF16) { return __uint_as_float((unsigned)x << 16); }
__device__ __forceinline__ float to_float(_Float16 x, F16) { return (float)x; }
__device__ __forceinline__ float from_float(float x, F32) { return x; }
__device__ __forceinline__ uint16_t from_float(float x, BF16) {
  const __bf16 b = (__bf16)x;  // round to nearest even
  return __builtin_bit_cast(uint16_t, b);
}
__device__ __forceinline__ _Float16 from_float(float x, F16) { return (_Float16)x; }

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

template <class D>
struct alignas(16) Pack {
  typename D::type v[D::kVec];
};

// Rows on 16-byte boundaries (VEC) promise that to the compiler; others (an odd vocabulary, a column slice) only the alignment
// of their elements.  The memory pipeline takes a 16-byte access at either, so a whole group is one instruction in both.  Element
// by element, as it was, an instruction moved an eighth (fp32: a quarter) of the bytes: 3001 x 152063 bf16 forward 555 -> 187 us,
// backward 956 -> 296 (152064 columns: 141 and 283); 1500 x 152063 fp32 forward 217 -> 152, backward 566 -> 318 (140 and 298).
typedef unsigned u32x4_at4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4_at2_t __attribute__((ext_vector_type(4), aligned(2)));
template <class D, bool VEC>
struct Group {
  using type = std::conditional_t<VEC, u32x4_t, std::conditional_t<sizeof(typename D::type) == 4, u32x4_at4_t, u32x4_at2_t>>;
};

// A launch reads logits once.  STREAM: non-temporal, which is worth 7 % of HBM bandwidth over logits that no cache holds.
template <class D, bool VEC, bool STREAM>
__device__ __forceinline__ u32x4_t load_whole(const typename D::type* __restrict__ p) {
  const auto* const q = reinterpret_cast<const typename Group<D, VEC>::type*>(p);
  if constexpr (STREAM) return __builtin_nontemporal_load(q);
  else return *q;
}

// The ragged group a row ends in: elements at or beyond `cols` read as `fill`.
template <class D>
__device__ __forceinline__ void load_ragged(const typename D::type* __restrict__ row, int64_t c, int64_t cols,
                                            float fill, float (&x)[D::kVec]) {
#pragma unroll
  for (int e = 0; e < D::kVec; ++e) x[e] = (c + e < cols) ? to_float(row[c + e], D()) : fill;
}

template <class D, bool VEC>
__device__ __forceinline__ void store_group(typename D::type* __restrict__ row, int64_t c, int64_t cols,
                                            const float (&x)[D::kVec]) {
  if (c + D::kVec <= cols) {
    Pack<D> p;
#pragma unroll
    for (int e = 0; e < D::kVec; ++e) p.v[e] = from_float(x[e], D());
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, p), reinterpret_cast<typename Group<D, VEC>::type*>(row + c));
  } else {
#pragma unroll
    for (int e = 0; e < D::kVec; ++e)
      if (c + e < cols) row[c + e] = from_float(x[e], D());
  }
}

template <class D>
inline bool rows_vectorizable(const void* base, int64_t ld) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && (ld * (int64_t)sizeof(typename D::type)) % 16 == 0;
}

// Rows of the logits that are read with plain loads, which leave them in the 256 MB memory-side cache for the next pass over the
// same logits (log-probs, entropies and the two gradients are four).  Logits that about fit are all read so; of larger ones the
// forward pass reads the first 224 MB so, the rest with the non-temporal hint, which does not displace them.  The four passes, all
// non-temporal and so, us: bf16 300 x 152064 (91 MB) 130 -> 117, 500 rows 180 -> 160, 800 rows (243 MB) 280 -> 258, 1000 rows
// (304 MB) 334 -> 327, 1500 rows 501 -> 493, 3001 rows 985 -> 976; fp32 400 x 151936 (243 MB) 280 -> 240, 500 rows 334 -> 312,
// 1500 rows 1030 -> 1013.  With plain loads for everything 1500 rows bf16 take 513, 3001 rows 1023; with the choice inside the
// backward kernel, whose small workgroups it delays, 800 rows 296.
constexpr int64_t kFittingBytes = 320ll << 20, kCachedBytes = 224ll << 20;
inline int64_t cached_rows(int64_t n_rows, int64_t ld, size_t element) {
  const int64_t pitch = ld * (int64_t)element;
  return n_rows * pitch <= kFittingBytes ? n_rows : kCachedBytes / pitch;
}

inline int check_rows(const char* what, const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t ld) {
  VAMD_REQUIRE(logits != nullptr, "%s: null logits", what);
  VAMD_REQUIRE(dtype >= VAMD_DT_F32 && dtype <= VAMD_DT_F16, "%s: unknown element type code %d", what, dtype);
  VAMD_REQUIRE(n_rows > 0 && vocab > 0 && ld >= vocab, "%s: bad shape rows=%lld vocab=%lld ld=%lld", what,
               (long long)n_rows, (long long)vocab, (long long)ld);
  VAMD_REQUIRE(n_rows < (1ll << 31), "%s: too many rows", what);
  return VAMD_OK;
}

}  // namespace
}  // namespace vamd

#define VAMD_DTYPE_DISPATCH(code, D, ...)                  \
  switch (code) {                                          \
    case VAMD_DT_F32: { using D = F32; __VA_ARGS__; } break;   \
    case VAMD_DT_BF16: { using D = BF16; __VA_ARGS__; } break; \
    default: { using D = F16; __VA_ARGS__; } break;            \
  }
