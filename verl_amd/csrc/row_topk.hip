// The k largest logits of a row as log-probabilities, beside the log-probability of a given token and the entropy; and the
// divergence of a row's softmax from a teacher's k most likely tokens.  Both with their gradients.
//
// With y = z log2(e) / T, m = max y and s = sum 2^(y - m):  log q_j = ((y_j - m) - log2 s) ln 2.
//   top alternatives: the k largest z, the lowest column first among equals (-0 equals 0; a NaN is below everything, and every
//     log-probability of its row is NaN); entropy = lse - sum q z / T, where q = 0 adds nothing, so that logits of -inf are allowed
//   divergence, over a teacher's tokens i_k with log-probabilities t_k, p = exp(t_k), q = q at i_k, b = beta:
//     forward KL  sum p (t - log q)                                  c_k = -p
//     reverse KL  sum q (log q - t)                                  c_k = q (log q - t + 1)
//     JSD         b sum p (t - log w) + (1 - b) sum q (log q - log w)   c_k = (1 - b) q (log q - log w),  w = b p + (1 - b) q
//     where c_k = d loss / d log q_k, and an entry outside [0, vocab), or whose t is -inf, adds nothing
//   gradients: d z_j = (sum_k g_k [j = i_k] - q_j sum_k g_k) / T for upstream gradients g_k of log q at i_k, and for the entropy
//     -g q_j (z_j - mean) / T^2
// Bound by HBM: the logits are read once, backward read and written once.
#include "common.h"
#include "divergence.h"
#include "head_pick.h"
#include "logit_rows.h"

namespace vamd {
namespace {

constexpr int kNarrow = 256, kMiddle = 512, kWide = 1024;  // threads per workgroup
constexpr int kMaxK = VAMD_TOPK_MAX;
constexpr float kInf = __builtin_huge_valf();

struct Softmax {
  float m, s, sz;  // max y, sum 2^(y - m), sum 2^(y - m) z
};
// A row's state as its users have it: of z - shift, where shift is 0 but for rows of lowest().
struct RowState : Softmax {
  float shift;
};
__device__ __forceinline__ void merge(Softmax& a, const Softmax& b) {
  const float m = fmaxf(a.m, b.m);
  const float x = __builtin_amdgcn_exp2f(a.m - m), y = __builtin_amdgcn_exp2f(b.m - m);
  a = Softmax{m, a.s * x + b.s * y, a.sz * x + b.sz * y};
}
// log q of logit z; the lowest values of a type, which masks are made of, would overflow as y
__device__ __forceinline__ float log_q(float z, float scale2, const RowState& r) {
  const float log2_s = log2f(r.s);
  z -= r.shift;
  return z < -1.0e30f ? fmaf(z, scale2 * kLn2, -(r.m + log2_s) * kLn2) : (fmaf(z, scale2, -r.m) - log2_s) * kLn2;
}

// what another lane of the row of 16 holds
template <int CTRL>
__device__ __forceinline__ float exchanged(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, false));
}

// A thread's kInFlight groups of logits into its state; returns what they add to sz.  The trip's terms are summed apart and added to
// the state once: one after the other, the few hundred terms of a thread lose a digit of the sums.  SUM_Z: whether sz is wanted.
template <bool SUM_Z, int G>
__device__ __forceinline__ float add_trip(const float (&x)[kInFlight][G], float hi, float scale2, Softmax& st) {
  const float y = hi * scale2;
  if (y > st.m) {
    const float resc = __builtin_amdgcn_exp2f(st.m - y);
    st.s *= resc;
    st.sz *= resc;
    st.m = y;
  }
  float s[kInFlight], sz[kInFlight];
#pragma unroll
  for (int u = 0; u < kInFlight; ++u) {
    s[u] = sz[u] = 0.f;
#pragma unroll
    for (int e = 0; e < G; ++e) {
      const float ex = __builtin_amdgcn_exp2f(fmaf(x[u][e], scale2, -st.m));
      s[u] += ex;
      if (SUM_Z) sz[u] = fmaf(ex, x[u][e], sz[u]);
    }
  }
  static_assert(kInFlight == 4, "the sums below");
  st.s += (s[0] + s[1]) + (s[2] + s[3]);
  return (sz[0] + sz[1]) + (sz[2] + sz[3]);
}
// The same sz where a logit is -inf, which adds 0 and not 0 x -inf, or NaN; read again, so that the trip's logits need not be held.
template <class D>
__device__ __forceinline__ float sum_with_masked(const typename D::type* row, int64_t c, int64_t stride, int64_t end, float scale2,
                                                 float m) {
  float sz = 0.f;
#pragma unroll 1
  for (int u = 0; u < kInFlight; ++u, c += stride)
#pragma unroll 1
    for (int e = 0; e < D::kVec; ++e) {
      const float z = c + e < end ? to_float(row[c + e], D()) : -kInf;
      sz = fmaf(__builtin_amdgcn_exp2f(fmaf(z, scale2, -m)), z == -kInf ? 0.f : z, sz);
    }
  return sz;
}

// What the walk leaves of a thread's trip in LDS: the largest logit, or for 16-bit types, which lose nothing by it, those of the first
// and of the last two loads, side by side.  A smaller group is less to read again (its loads lie in lines of their own); one of 64
// bytes in a row, over the lanes of a quad, took ten operations a trip: 4096 x 152064 bf16 k = 5 207 -> 221 us.
template <class D>
struct GroupWord {
  static constexpr int kHalves = sizeof(typename D::type) == 4 ? 1 : 2, kLoads = kInFlight / kHalves;
  static __device__ __forceinline__ unsigned pack(float a, float b) {
    if constexpr (std::is_same_v<D, F32>) return __float_as_uint(fmaxf(a, b));
    else if constexpr (std::is_same_v<D, BF16>) return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    else return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(a, b));
  }
  static __device__ __forceinline__ float half(unsigned word, int i) {
    if constexpr (std::is_same_v<D, F32>) return __uint_as_float(word);
    else if constexpr (std::is_same_v<D, BF16>) return __uint_as_float(i ? word & 0xffff0000u : word << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(i ? word >> 16 : word));
  }
};

// One thread's part of the columns [begin, end).  TOP: beside the softmax state a word of every `span` trips goes to LDS; `best` is the
// thread's largest logit.
template <class D, bool VEC, bool STREAM, int NT, bool TOP, bool SUM_Z>
__device__ __forceinline__ void walk(const typename D::type* __restrict__ row, int64_t begin, int64_t end, float scale2,
                                     int span, Softmax& st, float& best, unsigned* groups) {
  constexpr int G = D::kVec;
  constexpr int64_t stride = (int64_t)NT * G, trip = stride * kInFlight;
  float held[2] = {-kInf, -kInf};
  int left = span, slot = threadIdx.x;
  best = -kInf;
  st = Softmax{kNegBig, 0.f, 0.f};
  // the trip's largest logit
  const auto highest = [&](const float (&x)[kInFlight][G], bool last) {
    float h[2] = {-kInf, -kInf};
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
#pragma unroll
      for (int e = 0; e < G; ++e) h[u / (kInFlight / 2)] = fmaxf(h[u / (kInFlight / 2)], x[u][e]);
    const float hi = fmaxf(h[0], h[1]);
    if constexpr (TOP) {
      best = fmaxf(best, hi);
      held[0] = fmaxf(held[0], h[0]);
      held[1] = fmaxf(held[1], h[1]);
      if (--left == 0 || last) {
        groups[slot] = GroupWord<D>::pack(held[0], held[1]);
        held[0] = held[1] = -kInf;
        slot += NT;
        left = span;
      }
    }
    return hi;
  };
  const auto add = [&](const float (&x)[kInFlight][G], float hi, int64_t at) {
    float sz = add_trip<SUM_Z>(x, hi, scale2, st);
    if constexpr (SUM_Z) {
      if (__builtin_expect(sz != sz, 0)) sz = sum_with_masked<D>(row, at + (int)threadIdx.x * G, stride, end, scale2, st.m);
      st.sz += sz;
    }
  };
  int64_t base = begin;
  for (; base + trip <= end; base += trip) {
    u32x4_t raw[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) raw[u] = load_whole<D, VEC, STREAM>(row + base + u * stride + (int)threadIdx.x * G);
    float x[kInFlight][G];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const Pack<D> p = __builtin_bit_cast(Pack<D>, raw[u]);
#pragma unroll
      for (int e = 0; e < G; ++e) x[u][e] = to_float(p.v[e], D());
    }
    const float hi = highest(x, base + trip >= end);
    add(x, hi, base);
  }
  if (base < end) {  // the rest: missing logits are -inf, and kNegBig where they are summed
    const int left_here = (int)(end - base) - (int)threadIdx.x * G;
    u32x4_t raw[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)  // all of them requested first
      if (left_here - u * (int)stride >= G) raw[u] = load_whole<D, VEC, STREAM>(row + base + u * stride + (int)threadIdx.x * G);
    float x[kInFlight][G];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int n = left_here - u * (int)stride;
      if (n >= G) {
        const Pack<D> p = __builtin_bit_cast(Pack<D>, raw[u]);
#pragma unroll
        for (int e = 0; e < G; ++e) x[u][e] = to_float(p.v[e], D());
      } else {
#pragma unroll
        for (int e = 0; e < G; ++e) x[u][e] = -kInf;
        if (n > 0) load_ragged<D>(row, end - n, end, -kInf, x[u]);
      }
    }
    const float hi = highest(x, true);
    bool any = false;  // logits other than -inf: without one m may still be kNegBig, and kNegBig no small exponent
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
#pragma unroll
      for (int e = 0; e < G; ++e) {
        any = any || x[u][e] != -kInf;
        if (e >= left_here - u * (int)stride) x[u][e] = kNegBig;
      }
    if (any) add(x, hi, base);
  }
}

// the wavefront's state in every lane: within rows of 16 lanes by moves inside the vector ALU, then the four rows
template <int CTRL>
__device__ __forceinline__ void merge_exchanged(Softmax& st) {
  merge(st, Softmax{exchanged<CTRL>(st.m), exchanged<CTRL>(st.s), exchanged<CTRL>(st.sz)});
}
__device__ __forceinline__ Softmax in_lane(const Softmax& st, int lane) {
  const auto read = [lane](float x) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane)); };
  return Softmax{read(st.m), read(st.s), read(st.sz)};
}
__device__ __forceinline__ void merge_wave(Softmax& st) {
  merge_exchanged<0xB1>(st);   // lane ^ 1
  merge_exchanged<0x4E>(st);   // lane ^ 2
  merge_exchanged<0x141>(st);  // the other half of 8
  merge_exchanged<0x140>(st);  // the other half of 16
  Softmax a = in_lane(st, 0), b = in_lane(st, 32);
  merge(a, in_lane(st, 16));
  merge(b, in_lane(st, 48));
  merge(a, b);
  st = a;
}

// The state of a row without a logit that a walk can tell from -inf (s is 0: every y lies below kNegBig), taken from its largest
// logit: a row masked throughout with the lowest value of its type is uniform, one of -inf is NaN.  Every thread of the workgroup
// comes here.
template <class D, int NT>
__device__ __forceinline__ RowState lowest(const typename D::type* __restrict__ row, int64_t cols, float scale2) {
  __shared__ float red[3][NT / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  float hi = -kInf, s = 0.f, sz = 0.f;
#pragma unroll 1
  for (int64_t c = threadIdx.x; c < cols; c += NT) hi = fmaxf(hi, to_float(row[c], D()));
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) hi = fmaxf(hi, __shfl_xor(hi, off, 64));
  if (lane == 0) red[0][w] = hi;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NT / 64; ++j) hi = fmaxf(hi, red[0][j]);
#pragma unroll 1
  for (int64_t c = threadIdx.x; c < cols; c += NT) {
    const float z = to_float(row[c], D()) - hi;
    const float ex = __builtin_amdgcn_exp2f(z * scale2);
    s += ex;
    sz = fmaf(ex, ex == 0.f ? 0.f : z, sz);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    s += __shfl_xor(s, off, 64);
    sz += __shfl_xor(sz, off, 64);
  }
  if (lane == 0) {
    red[1][w] = s;
    red[2][w] = sz;
  }
  __syncthreads();
  s = sz = 0.f;
#pragma unroll
  for (int j = 0; j < NT / 64; ++j) {
    s += red[1][j];
    sz += red[2][j];
  }
  return RowState{{0.f, s, sz}, hi};
}

// ---- the k largest of a range of a row ------------------------------------------------------------------------
// A logit as a number that orders like it, -0 as 0, NaN lowest; with its column below it, so that the largest comes first and
// among equals the lowest column, and no two are the same.
__device__ __forceinline__ unsigned order_of(float z) {
  const unsigned b = __float_as_uint(z + 0.f);
  return z != z ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
constexpr unsigned kOrderOfMinusInf = 0x007fffffu;
__device__ __forceinline__ float logit_of(unsigned order) {
  return order == 0u ? __builtin_nanf("") : __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ uint64_t entry_of(unsigned order, int64_t col) {
  return (uint64_t)order << 32 | (0xffffffffu - (unsigned)col);
}
__device__ __forceinline__ unsigned order_in(uint64_t entry) { return (unsigned)(entry >> 32); }
__device__ __forceinline__ int64_t column_in(uint64_t entry) { return (int64_t)(0xffffffffu - (unsigned)entry); }

// The walk leaves the maximum of every group in LDS (at most kGroupBytes; a row of 152064 bf16 has 4864 words for 9728 groups of
// 16 logits).  The k-th largest of the threads' own maxima is a value that at least k logits reach; only groups that reach it can hold
// one of the k largest, and these, about k of them, are read again: k x 2 lines instead of the row.  What reaches
// the value there, a little more than k logits, is ranked by counting.  Where that list would be too long (many equal logits)
// the order of the k-th largest is found digit by digit in passes over the row, which is right for any values.
constexpr int kGroupBytes = 20 * 1024, kGroupList = 512, kCandidates = 1024;

template <int NT>
struct PickLds {
  unsigned top[NT];  // the threads' maxima; later the digit counts
  int group[kGroupList];
  float red[3][NT / 64];
  Softmax whole;
  unsigned least;
  int groups, candidates, digit, above, wave[NT / 64];
};

// the state of the whole workgroup, and for pick() the value that at least k logits reach, in `least`
template <class D, int NT>
__device__ __forceinline__ void meet(PickLds<NT>& lds, Softmax st, float best, int k) {
  // bits below it cannot tell two logits of the type apart (fp32: change the value by less than 2^-14)
  constexpr int kLowBit = std::is_same_v<D, BF16> ? 16 : std::is_same_v<D, F16> ? 13 : 9;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int role = (w + (int)blockIdx.x) % (NT / 64);  // every SIMD has one wavefront of each workgroup, so they take turns
  merge_wave(st);
  if (lane == 0) {
    lds.red[0][w] = st.m;
    lds.red[1][w] = st.s;
    lds.red[2][w] = st.sz;
  }
  lds.top[threadIdx.x] = order_of(best);
  if (threadIdx.x == 0) lds.groups = lds.candidates = 0;
  __syncthreads();
  if (role == 1) {
    Softmax all{lds.red[0][0], lds.red[1][0], lds.red[2][0]};
#pragma unroll
    for (int j = 1; j < NT / 64; ++j) merge(all, Softmax{lds.red[0][j], lds.red[1][j], lds.red[2][j]});
    if (lane == 0) lds.whole = all;
  } else if (role == 0) {
    constexpr int P = NT / 64;
    unsigned mine[P];
#pragma unroll
    for (int j = 0; j < P; ++j) mine[j] = lds.top[j * 64 + lane];
    const auto reach = [&](unsigned order) {
      int n = 0;
#pragma unroll
      for (int j = 0; j < P; ++j) n += __popcll(__ballot(mine[j] >= order));
      return n;
    };
    unsigned least = kOrderOfMinusInf + 1;  // fewer than k threads with a finite logit: every finite one
    if (reach(least) >= k) {
      unsigned order = 0;
      for (int bit = 31; bit >= kLowBit; --bit)
        if (reach(order | 1u << bit) >= k) order |= 1u << bit;
      if (order > least) least = order;
    }
    if (lane == 0) lds.least = least;
  }
  __syncthreads();
}

// emit(rank, entry) for each entry of the list that is among its k largest.  A short list is ranked by counting, which reads it once
// per wavefront of entries (all lanes the same words, at the speed of 64 different ones); a longer one is sorted, by exchanges
// between entries a power of two apart: 64 x 152064 bf16, k = 256, lists of 400 to 900, 120 us by counting.
// The list has room for the next power of two; every thread comes here with the list complete.
constexpr int kCountedList = 192;
template <int NT, class Emit>
__device__ __forceinline__ void rank_list(uint64_t* list, int n, int k, Emit&& emit) {
  if (n <= kCountedList) {
    for (int j = (threadIdx.x + 64u * blockIdx.x) % NT; j < n; j += NT) {
      const uint64_t mine = list[j];
      int rank = 0, i = 0;
      for (; i + 8 <= n; i += 8) {  // eight reads in flight
#pragma unroll
        for (int u = 0; u < 8; ++u) rank += list[i + u] > mine;
      }
      for (; i < n; ++i) rank += list[i] > mine;
      if (rank < k) emit(rank, mine);
    }
    return;
  }
  int size = 256;
  while (size < n) size *= 2;
  for (int j = n + threadIdx.x; j < size; j += NT) list[j] = 0;
  __syncthreads();
  for (int run = 2; run <= size; run *= 2)
    for (int apart = run / 2; apart > 0; apart /= 2) {
      for (int t = threadIdx.x; t < size / 2; t += NT) {
        const int i = (t & ~(apart - 1)) << 1 | (t & (apart - 1)), j = i + apart;
        const uint64_t x = list[i], y = list[j];
        if ((x < y) == ((i & run) == 0)) {
          list[i] = y;
          list[j] = x;
        }
      }
      __syncthreads();
    }
  for (int j = threadIdx.x; j < n && j < k; j += NT) emit(j, list[j]);
}

// emit(rank, entry) for the first `need` columns of the range whose logit is of this order, from `rank` on; returns how many
template <class D, int NT, class Emit>
__device__ int rank_equal(PickLds<NT>& lds, const typename D::type* __restrict__ row, int64_t begin, int64_t end,
                          unsigned order, int need, int rank, Emit&& emit) {
  constexpr int G = D::kVec;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int found = 0;
  for (int64_t base = begin; base < end && found < need; base += (int64_t)NT * G) {
    const int64_t c = base + (int64_t)threadIdx.x * G;
    unsigned here = 0;
#pragma unroll
    for (int e = 0; e < G; ++e)
      if (c + e < end && order_of(to_float(row[c + e], D())) == order) here |= 1u << e;
    const int n = __popc(here);
    int before = n;  // in this and lower lanes
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int x = __shfl_up(before, off, 64);
      if (lane >= off) before += x;
    }
    __syncthreads();
    if (lane == 63) lds.wave[w] = before;
    __syncthreads();
    int place = found + before - n, all = found;
    for (int j = 0; j < NT / 64; ++j) {
      if (j < w) place += lds.wave[j];
      all += lds.wave[j];
    }
#pragma unroll
    for (int e = 0; e < G; ++e)
      if (here >> e & 1u) {
        if (place < need) emit(rank + place, entry_of(order, c + e));
        ++place;
      }
    found = all;
  }
  return found < need ? found : need;
}

// by digits: passes over the range, for any values
template <class D, int NT, class Emit>
__device__ void pick_by_digits(PickLds<NT>& lds, uint64_t* list, const typename D::type* __restrict__ row, int64_t begin,
                               int64_t end, int k, Emit&& emit) {
  const int kk = (int)(end - begin < k ? end - begin : k);
  unsigned order = 0, known = 0;
  int need = kk;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int j = threadIdx.x; j < 256; j += NT) lds.top[j] = 0;
    __syncthreads();
    for (int64_t c = begin + threadIdx.x; c < end; c += NT) {
      const unsigned o = order_of(to_float(row[c], D()));
      if ((o & known) != order) continue;
      const unsigned digit = o >> shift & 255u;
      // one addition for a wavefront of equal digits
      const uint64_t active = __ballot(true);
      if (__ballot(digit == (unsigned)__builtin_amdgcn_readfirstlane((int)digit)) == active) {
        if ((int)(threadIdx.x & 63) == __ffsll((unsigned long long)active) - 1) atomicAdd(&lds.top[digit], (unsigned)__popcll(active));
      } else {
        atomicAdd(&lds.top[digit], 1u);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int above = 0, digit = 255;
      while (digit > 0 && above + (int)lds.top[digit] < need) above += (int)lds.top[digit--];
      lds.digit = digit;
      lds.above = above;
    }
    __syncthreads();
    order |= (unsigned)lds.digit << shift;
    known |= 255u << shift;
    need -= lds.above;
  }
  // kk - need logits are above the k-th largest, `need` of its equals belong to the k
  if (threadIdx.x == 0) lds.candidates = 0;
  __syncthreads();
  for (int64_t c = begin + threadIdx.x; c < end; c += NT) {
    const unsigned o = order_of(to_float(row[c], D()));
    if (o > order) list[atomicAdd(&lds.candidates, 1)] = entry_of(o, c);
  }
  __syncthreads();
  rank_list<NT>(list, kk - need, k, emit);
  rank_equal<D, NT>(lds, row, begin, end, order, need, kk - need, emit);
}

// Where the logits of a group lie that the walk has left a maximum of: pieces() x 16 bytes.
template <class D, int NT>
struct WalkLayout {
  using Word = GroupWord<D>;
  int64_t begin;
  int words, span;
  __device__ __forceinline__ int pieces() const { return Word::kLoads * span; }
  __device__ __forceinline__ int64_t column(int group, int piece) const {
    const int slot = group / Word::kHalves;
    const int64_t load = (int64_t)(slot / NT * span + piece / Word::kLoads) * kInFlight + group % Word::kHalves * Word::kLoads + piece % Word::kLoads;
    return begin + (load * NT + slot % NT) * D::kVec;
  }
};
// Of a tile of the head's epilogue (HeadPickArgs).
struct TileLayout {
  using Word = GroupWord<F32>;
  int words;
  __device__ __forceinline__ int pieces() const { return 8; }
  __device__ __forceinline__ int64_t column(int group, int piece) const {
    return 256 * (int64_t)(group >> 3) + 128 * (group >> 2 & 1) + 4 * (group & 3) + 16 * piece;
  }
};

// emit(rank, entry) once for every rank below k that the range has, by any thread.  `groups`: the maxima in LDS, which has room for
// kCandidates entries; they are overwritten.  meet() has run.
template <class D, bool VEC, int NT, class Layout, class Emit>
__device__ __forceinline__ void pick(PickLds<NT>& lds, unsigned* groups, const Layout& layout,
                                     const typename D::type* __restrict__ row, int64_t begin, int64_t end, int k, float best,
                                     Emit&& emit) {
  using Word = typename Layout::Word;
  constexpr int G = D::kVec, H = Word::kHalves;
  const float least = logit_of(lds.least);
  const bool all_finite = lds.least == kOrderOfMinusInf + 1;
  if (best >= least)
    for (int slot = threadIdx.x; slot < layout.words; slot += NT) {
      const unsigned word = groups[slot];
#pragma unroll
      for (int i = 0; i < H; ++i)
        if (Word::half(word, i) >= least) {
          const int at = atomicAdd(&lds.groups, 1);
          if (at < kGroupList) lds.group[at] = slot * H + i;
        }
    }
  __syncthreads();
  uint64_t* const list = reinterpret_cast<uint64_t*>(groups);
  const int pieces = layout.pieces(), n_groups = lds.groups;
  if (n_groups <= kGroupList) {
    for (int j = threadIdx.x; j < n_groups * pieces; j += NT) {
      const int64_t c = layout.column(lds.group[j / pieces], j % pieces);
      float x[G];
      if (c + G <= end) {
        const Pack<D> p = __builtin_bit_cast(Pack<D>, load_whole<D, VEC, false>(row + c));
#pragma unroll
        for (int e = 0; e < G; ++e) x[e] = to_float(p.v[e], D());
      } else {
        load_ragged<D>(row, c, end, -kInf, x);
      }
#pragma unroll
      for (int e = 0; e < G; ++e)
        if (x[e] >= least) {
          const int at = atomicAdd(&lds.candidates, 1);
          if (at < kCandidates) list[at] = entry_of(order_of(x[e]), c + e);
        }
    }
    __syncthreads();
    const int n = lds.candidates;
    if (n <= kCandidates && (n >= k || all_finite)) {
      rank_list<NT>(list, n, k, emit);
      if (n < k) {
        // the others are -inf, and then NaN, in the order of their columns
        const int64_t more = end - begin - n;
        const int need = (int)(more < k - n ? more : k - n);
        const int got = rank_equal<D, NT>(lds, row, begin, end, kOrderOfMinusInf, need, n, emit);
        rank_equal<D, NT>(lds, row, begin, end, 0u, need - got, n + got, emit);
      }
      return;
    }
  }
  pick_by_digits<D, NT>(lds, list, row, begin, end, k, emit);
}

struct TopkArgs {
  const void* logits;
  int64_t ld, cols;
  const int64_t* labels;
  int k, span;
  float scale2, rcp_t;
  float* logprobs;
  float* entropy;
  float* top;      // [rows][k]
  int64_t* index;  // [rows][k]
  float4* stats;   // m, 1 / s, mean of z - shift, shift
  int64_t cached_rows;
  int splits;  // of a row; more than one: each leaves its state and its k largest, for row_topk_join_kernel
  int64_t split_cols;
  float4* part_state;     // [rows][splits]
  uint64_t* part_entry;  // [rows][splits][k], largest first, 0 where there are fewer
};

struct RowResult {
  const TopkArgs& a;
  int64_t r;
  RowState st;
  __device__ __forceinline__ void operator()(int rank, uint64_t entry) const {
    a.top[r * a.k + rank] = log_q(logit_of(order_in(entry)), a.scale2, st);
    a.index[r * a.k + rank] = column_in(entry);
  }
  template <class D>
  __device__ __forceinline__ void scalars(const typename D::type* __restrict__ row) const {
    const float lse = (st.m + log2f(st.s)) * kLn2, mean = st.sz / st.s;
    if (a.entropy) a.entropy[r] = fmaf(-mean, a.rcp_t, lse);
    if (a.stats) a.stats[r] = make_float4(st.m, 1.f / st.s, mean, st.shift);
    if (a.logprobs) {  // a label outside [0, cols) reads nothing and yields 0
      const int64_t label = a.labels[r];
      a.logprobs[r] = label >= 0 && label < a.cols ? log_q(to_float(row[label], D()), a.scale2, st) : 0.f;
    }
  }
};

template <class D, bool VEC, int NT>
__global__ __launch_bounds__(NT) void row_topk_kernel(TopkArgs a) {
  using T = typename D::type;
  extern __shared__ __attribute__((aligned(16))) unsigned groups[];
  __shared__ PickLds<NT> lds;
  const int64_t r = a.splits > 1 ? blockIdx.x / a.splits : blockIdx.x;
  const int split = a.splits > 1 ? (int)(blockIdx.x % a.splits) : 0;
  const int64_t begin = split * a.split_cols, end = begin + a.split_cols < a.cols ? begin + a.split_cols : a.cols;
  const T* __restrict__ row = static_cast<const T*>(a.logits) + r * a.ld;
  Softmax st;
  float best;
  if (r < a.cached_rows) walk<D, VEC, false, NT, true, true>(row, begin, end, a.scale2, a.span, st, best, groups);
  else walk<D, VEC, true, NT, true, true>(row, begin, end, a.scale2, a.span, st, best, groups);
  meet<D, NT>(lds, st, best, a.k);
  st = lds.whole;
  constexpr int64_t trip = (int64_t)NT * D::kVec * kInFlight;
  const int trips = (int)((end - begin + trip - 1) / trip);
  const WalkLayout<D, NT> layout{begin, (trips + a.span - 1) / a.span * NT, a.span};
  if (a.splits > 1) {
    const int64_t part = r * a.splits + split;
    uint64_t* const out = a.part_entry + part * a.k;
    pick<D, VEC, NT>(lds, groups, layout, row, begin, end, a.k, best, [&](int rank, uint64_t entry) { out[rank] = entry; });
    for (int64_t j = end - begin + threadIdx.x; j < a.k; j += NT) out[j] = 0;
    if (threadIdx.x == 0) a.part_state[part] = make_float4(st.m, st.s, st.sz, 0.f);
  } else {
    RowState state{st, 0.f};
    if (st.s == 0.f) state = lowest<D, NT>(row, a.cols, a.scale2);
    const RowResult result{a, r, state};
    pick<D, VEC, NT>(lds, groups, layout, row, begin, end, a.k, best, result);
    if (threadIdx.x == 0) result.template scalars<D>(row);
  }
}

// The k largest of a token's logits that the head has written out.
template <int NT>
__global__ __launch_bounds__(NT) void head_pick_kernel(HeadPickArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned groups[];
  __shared__ PickLds<NT> lds;
  const int64_t tok = blockIdx.x;
  const float* __restrict__ row = a.z + tok * a.z_ld;
  const float* __restrict__ maxima = a.group_max + tok * a.groups;
  float best = -kInf;
  for (int j = threadIdx.x; j < a.groups; j += NT) {
    const float x = maxima[j];
    groups[j] = __float_as_uint(x);
    best = fmaxf(best, x);
  }
  meet<F32, NT>(lds, Softmax{kNegBig, 0.f, 0.f}, best, a.k);
  const float lse = a.lse[tok];
  pick<F32, true, NT>(lds, groups, TileLayout{a.groups}, row, 0, a.vocab, a.k, best, [&](int rank, uint64_t entry) {
    a.top[tok * a.k + rank] = fmaf(logit_of(order_in(entry)), a.rcp_t, -lse);
    a.index[tok * a.k + rank] = column_in(entry);
  });
}

// A row's splits: of S lists that fall, the smallest of their ceil(k / S)-th entries is a value that at least k entries reach, and so is
// any list's k-th; the entries that reach the larger of the two, usually a few times k, are ranked by counting.
template <class D>
__global__ __launch_bounds__(kNarrow) void row_topk_join_kernel(TopkArgs a) {
  extern __shared__ __attribute__((aligned(16))) unsigned groups[];
  uint64_t* const list = reinterpret_cast<uint64_t*>(groups);
  __shared__ Softmax whole;
  __shared__ uint64_t reach;
  __shared__ int found;
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = a.splits * a.k, place = (a.k + a.splits - 1) / a.splits - 1;
  const uint64_t* const parts = a.part_entry + r * n;
  if (threadIdx.x == 0) found = 0;
  if (w == 0) {
    Softmax st{kNegBig, 0.f, 0.f};
    for (int j = lane; j < a.splits; j += 64) {
      const float4 x = a.part_state[r * a.splits + j];
      merge(st, Softmax{x.x, x.y, x.z});
    }
    merge_wave(st);
    if (lane == 0) whole = st;
  } else if (w == 1) {
    uint64_t least = ~0ull, last = 0;
    for (int j = lane; j < a.splits; j += 64) {
      const uint64_t x = parts[j * a.k + place], y = parts[j * a.k + a.k - 1];
      least = x < least ? x : least;
      last = y > last ? y : last;
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      const uint64_t x = __shfl_xor(least, off, 64), y = __shfl_xor(last, off, 64);
      least = x < least ? x : least;
      last = y > last ? y : last;
    }
    least = last > least ? last : least;
    if (lane == 0) reach = least > 0 ? least : 1;  // (0: no entry)
  }
  __syncthreads();
  const uint64_t least = reach;
  for (int j = threadIdx.x; j < n; j += kNarrow) {
    const uint64_t x = parts[j];
    if (x >= least) list[atomicAdd(&found, 1)] = x;
  }
  __syncthreads();
  const auto* const row = static_cast<const typename D::type*>(a.logits) + r * a.ld;
  RowState state{whole, 0.f};
  if (whole.s == 0.f) state = lowest<D, kNarrow>(row, a.cols, a.scale2);
  const RowResult result{a, r, state};
  rank_list<kNarrow>(list, found, a.k, result);
  if (threadIdx.x == 0) result.template scalars<D>(row);
}

// ---- divergence from a teacher's tokens -----------------------------------------------------------------------
// Entries of a gradient by column, equal columns in their order, those that do not count last; and the first one in each chunk of columns
// that a workgroup of the backward pass takes.  Where a row has more entries than a wavefront looks through at once.
struct Sorted {
  int* column;  // [rows][k]; null: not to be sorted
  float* grad;  // [rows][k]
  int* first;   // [rows][chunks + 1]
  int chunks, chunk_cols;
};
constexpr int kUnsortedEntries = 64;
constexpr int kNoEntry = 0x7fffffff;
// Thread t < k has entry t.  Every thread comes here.
template <int NT>
__device__ __forceinline__ void sort_entries(const Sorted& to, int64_t r, int k, int mine, float grad) {
  __shared__ int column[kMaxK], sorted[kMaxK];
  const int t = threadIdx.x;
  if (t < k) column[t] = mine;
  __syncthreads();
  if (t < k) {
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < k; ++i) rank += column[i] < mine || (column[i] == mine && i < t);
    sorted[rank] = mine;
    to.column[r * k + rank] = mine;
    to.grad[r * k + rank] = grad;
  }
  __syncthreads();
  for (int c = t; c <= to.chunks; c += NT) {
    const int64_t from = (int64_t)c * to.chunk_cols;
    int lo = 0, hi = k;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (sorted[mid] < from) lo = mid + 1;
      else hi = mid;
    }
    to.first[r * (to.chunks + 1) + c] = lo;
  }
}

struct DivergenceArgs {
  const void* logits;
  int64_t ld, cols;
  const float* teacher;  // [rows][k] log-probabilities
  const int64_t* index;  // [rows][k]
  int k, kind;
  float beta, scale2;
  float* loss;
  float4* stats;  // m, 1 / s, sum of the slopes, shift; null without a backward pass
  float* slope;   // [rows][k], where the entries are few
  Sorted sorted;  // where they are many
  int64_t cached_rows;
};

template <class D, bool VEC, int NT>
__global__ __launch_bounds__(NT) void row_divergence_kernel(DivergenceArgs a) {
  using T = typename D::type;
  __shared__ float red[2][NT / 64];
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const T* __restrict__ row = static_cast<const T*>(a.logits) + r * a.ld;
  // requested before the walk: they are a chain of two trips behind it otherwise
  int64_t index = -1;
  float t = -kInf, z = 0.f;
  if ((int)threadIdx.x < a.k) {
    index = a.index[r * a.k + threadIdx.x];
    t = a.teacher[r * a.k + threadIdx.x];
    if (index >= 0 && index < a.cols && t != -kInf) z = to_float(row[index], D());
    else index = -1;
  }
  Softmax st;
  float best;
  if (r < a.cached_rows) walk<D, VEC, false, NT, false, false>(row, 0, a.cols, a.scale2, 1, st, best, nullptr);
  else walk<D, VEC, true, NT, false, false>(row, 0, a.cols, a.scale2, 1, st, best, nullptr);
  merge_wave(st);
  if (lane == 0) {
    red[0][w] = st.m;
    red[1][w] = st.s;
  }
  __syncthreads();
  st = Softmax{red[0][0], red[1][0], 0.f};
#pragma unroll
  for (int j = 1; j < NT / 64; ++j) merge(st, Softmax{red[0][j], red[1][j], 0.f});
  RowState state{st, 0.f};
  if (st.s == 0.f) state = lowest<D, NT>(row, a.cols, a.scale2);
  Term mine{0.f, 0.f};
  if (index >= 0) mine = divergence_term(a.kind, a.beta, t, log_q(z, a.scale2, state));
  if (a.slope && (int)threadIdx.x < a.k) a.slope[r * a.k + threadIdx.x] = mine.slope;
  if (a.sorted.column) sort_entries<NT>(a.sorted, r, a.k, index >= 0 ? (int)index : kNoEntry, mine.slope);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    mine.loss += __shfl_xor(mine.loss, off, 64);
    mine.slope += __shfl_xor(mine.slope, off, 64);
  }
  __syncthreads();
  if (lane == 0) {
    red[0][w] = mine.loss;
    red[1][w] = mine.slope;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    constexpr int W = kMaxK / 64;  // the wavefronts that hold entries
    float loss = 0.f, slope = 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      loss += red[0][j];
      slope += red[1][j];
    }
    a.loss[r] = loss;
    if (a.stats) a.stats[r] = make_float4(state.m, 1.f / state.s, slope, state.shift);
  }
}
static_assert(kMaxK <= kNarrow, "an entry per thread");

// ---- gradient --------------------------------------------------------------------------------------------------
// d z_j = sum_k scale g_k [j = i_k] / T + g_lp [j = label] / T - q_j (scale weight / T + g_ent (z_j - mean z) / T^2)
struct EntriesArgs {
  const void* logits;
  int64_t ld, cols;
  int chunks, k;
  const int64_t* index;    // [rows][k]; one outside [0, cols) matches nothing
  const float* grad;       // [rows][k]: g_k
  Sorted sorted;           // the same where there are more than kUnsortedEntries
  const float4* stats;     // m, 1 / s, ., shift
  const float* weight;     // [rows]: sum of all g; null: the third of stats
  const float* scale;      // [rows] or null (1)
  const int64_t* labels;   // with d_logprobs
  const float* d_logprobs;
  const float* d_entropy;  // with it the third of stats is the mean of z
  float scale2, rcp_t;
  void* out;
  int64_t ld_out;
};

// One workgroup per (row, chunk of kNarrow * G * F columns), as row_softmax_backward_kernel, whose comments say why.  An entry is added,
// in order, in the registers of the lane that holds its column, so that an index that comes twice counts twice and each gradient
// is rounded once.  Up to 64 entries every wavefront looks through all of the row's for its own: they come with the logits.  More
// are sorted first, and a workgroup reads its own, behind the place of the first.  4096 x 152064 bf16, forward and backward pass of the
// divergence, us: 64 entries 581, 65 (sorted) 592, 128 607, 256 636; with every wavefront looking through all of them, before the
// arithmetic below was trimmed, 5 entries 606, 64 618, 128 690, 256 850.
// ENTROPY: an entropy has an upstream gradient.  Bound by HBM (6.4 TB/s).  With the label's comparison and the entropy's terms at every
// element the vector ALU was 89 % busy, and the pass took 428 us with 64 entries, now 388.
template <class D, bool VEC, bool STREAM, bool SORTED, bool ENTROPY>
__global__ __launch_bounds__(kNarrow) void row_entries_backward_kernel(EntriesArgs a) {
  using T = typename D::type;
  constexpr int G = D::kVec, F = D::kBackwardLoads;
  const int64_t r = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x % a.chunks, lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const T* __restrict__ row = static_cast<const T*>(a.logits) + r * a.ld;
  T* __restrict__ out = static_cast<T*>(a.out) + r * a.ld_out;
  constexpr int stride = kNarrow * G;
  const int64_t first = (int64_t)chunk * stride * F, c0 = first + (int)threadIdx.x * G;
  u32x4_t raw[F];
#pragma unroll
  for (int u = 0; u < F; ++u) {
    const int64_t c = c0 + u * stride;
    if (c + G <= a.cols) raw[u] = load_whole<D, VEC, STREAM>(row + c);
  }
  const int64_t entries = r * a.k;
  // the column of the entry that the lane looks at, and its gradient (as they come: a conversion would wait for them here)
  std::conditional_t<SORTED, int, int64_t> column = -1;
  float grad = 0.f;
  if (!SORTED && lane < a.k) column = a.index[entries + lane];
  __builtin_amdgcn_sched_barrier(0);
  const float4 st = a.stats[r];
  int e_begin = 0, e_end = a.k;
  if constexpr (SORTED) {
    const int* const place = a.sorted.first + r * (a.sorted.chunks + 1) + chunk;
    e_begin = place[0];
    e_end = place[1];
    if (e_begin + lane < e_end) {  // requested before the logits are waited for
      column = a.sorted.column[entries + e_begin + lane];
      grad = a.sorted.grad[entries + e_begin + lane];
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  const float scale = (a.scale ? a.scale[r] : 1.f) * a.rcp_t;
  const int64_t label = a.d_logprobs ? a.labels[r] : -1;
  // a token that a loss masks out, whose slopes may be NaN
  const bool out_of_loss = a.scale && scale == 0.f;
  if (out_of_loss) e_end = e_begin;
  const float g0 = out_of_loss ? 0.f : scale * (a.weight ? a.weight[r] : st.z), g1 = ENTROPY ? a.d_entropy[r] * a.rcp_t * a.rcp_t : 0.f;
  const float u0 = g0 * st.y, u1 = g1 * st.y;
  // a row that no gradient comes to, whatever its logits are
  const bool none = g0 == 0.f && g1 == 0.f;
  float x[F][G];
#pragma unroll
  for (int u = 0; u < F; ++u) {
    const int64_t c = c0 + u * stride;
    if (c + G <= a.cols) {
      const Pack<D> p = __builtin_bit_cast(Pack<D>, raw[u]);
#pragma unroll
      for (int e = 0; e < G; ++e) x[u][e] = to_float(p.v[e], D());
    } else {
      load_ragged<D>(row, c, a.cols, 0.f, x[u]);
    }
    if (none) {
#pragma unroll
      for (int e = 0; e < G; ++e) x[u][e] = 0.f;
      continue;
    }
    if (st.w != 0.f) {
#pragma unroll
      for (int e = 0; e < G; ++e) x[u][e] -= st.w;
    }
#pragma unroll
    for (int e = 0; e < G; ++e) {
      const float z = x[u][e];
      const float ex = __builtin_amdgcn_exp2f(fmaf(z, a.scale2, -st.x));
      // a logit below -1e20 has a q of 0, which -inf would make a NaN
      x[u][e] = -ex * (ENTROPY ? fmaf(u1, fmaxf(z, -1.0e20f) - st.z, u0) : u0);
    }
  }
  // adds g to the column `at` of the chunk (what lies past the row is not stored)
  const auto add = [&](int at, float g) {
    const int mine = at / G % 64 == lane ? at / stride * G + at % G : -1;
#pragma unroll
    for (int u = 0; u < F; ++u)
#pragma unroll
      for (int e = 0; e < G; ++e) x[u][e] += mine == u * G + e ? g : 0.f;
  };
  const int64_t label_at = label - first;
  if (label_at >= 0 && label_at < stride * F && (int)label_at / G % kNarrow / 64 == w) add((int)label_at, a.d_logprobs[r] * a.rcp_t);
  for (int e0 = e_begin; e0 < e_end; e0 += 64) {
    if (SORTED && e0 > e_begin && e0 + lane < e_end) {
      column = a.sorted.column[entries + e0 + lane];
      grad = a.sorted.grad[entries + e0 + lane];
    }
    const int64_t at64 = (int64_t)column - first;
    const bool inside = e0 + lane < e_end && at64 >= 0 && at64 < stride * F;
    const int at = inside ? (int)at64 : 0;
    uint64_t hits = __ballot(inside && at / G % kNarrow / 64 == w);
    while (hits) {
      const int b = __ffsll((unsigned long long)hits) - 1;
      hits &= hits - 1;
      add(__builtin_amdgcn_readlane(at, b),
          (SORTED ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(grad), b)) : a.grad[entries + b]) * scale);
    }
  }
#pragma unroll
  for (int u = 0; u < F; ++u) {
    const int64_t c = c0 + u * stride;
    if (c < a.cols) store_group<D, VEC>(out, c, a.cols, x[u]);
  }
}

// What the backward pass of the alternatives needs first: weight[r], the sum of d_top[r] and of d_logprobs[r] where the label counts, and
// where there are many alternatives their order.
__global__ __launch_bounds__(kNarrow) void row_topk_prepare_kernel(const float* d_logprobs, const int64_t* labels, int64_t cols,
                                                                   const float* d_top, const int64_t* index, int k, float* weight,
                                                                   Sorted sorted) {
  __shared__ float red[kNarrow / 64];
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x;
  const float grad = t < k ? d_top[r * k + t] : 0.f;
  float sum = grad;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if ((t & 63) == 0) red[t >> 6] = sum;
  __syncthreads();
  if (t == 0) {
    sum = red[0] + red[1] + red[2] + red[3];
    if (d_logprobs && labels[r] >= 0 && labels[r] < cols) sum += d_logprobs[r];
    weight[r] = sum;
  }
  if (!sorted.column) return;
  const int64_t i = t < k ? index[r * k + t] : -1;
  sort_entries<kNarrow>(sorted, r, k, i >= 0 && i < cols ? (int)i : kNoEntry, grad);
}
static_assert(kMaxK <= kNarrow, "an entry per thread");

// ---- host side -------------------------------------------------------------------------------------------------
// The maxima of how many threads give the value that about k logits reach.  4096 x 152064 bf16, 256, 512 and 1024 threads, us:
// k = 65 228, 242 and 325, 128 257, 265 and 341, 160 286, 272 and 350, 256 (256 threads: every maximum is reached) 326 and 434.
int threads_for(int k) { return k <= 128 ? kNarrow : kMiddle; }

constexpr int kJoinEntries = 4096;  // 32 KB of LDS in row_topk_join_kernel; a power of two, which rank_list may need

struct TopkPlan {
  int threads, span, splits;
  int64_t split_cols, slots;  // slots: group maxima per workgroup
  size_t lds_bytes() const {
    const size_t list = kCandidates * sizeof(uint64_t), maxima = (size_t)slots * sizeof(unsigned);
    return maxima > list ? maxima : list;
  }
};
TopkPlan plan_topk(int64_t n_rows, int64_t vocab, int dtype, int k) {
  TopkPlan p;
  p.threads = threads_for(k);
  const int64_t trip = (int64_t)p.threads * (dtype == VAMD_DT_F32 ? 4 : 8) * kInFlight;
  int64_t trips = (vocab + trip - 1) / trip;
  // Few rows: a row is shared out over workgroups, at least a trip each, until there are two of 256 threads to a CU (two, three,
  // four and eight, us: 64 x 152064 bf16 k = 20 16.2, 16.6, 21.5 and 22.2, 200 rows 23.4, 23.4, 23.2 and 27.2, 32 rows 15.1, 17.0,
  // 17.1 and 16.9).
  const int64_t workgroups = (int64_t)device_cu_count() * 2 * kNarrow / p.threads;
  int64_t splits = workgroups / n_rows;
  if (splits > trips) splits = trips;
  if (splits > kJoinEntries / k) splits = kJoinEntries / k;
  if (splits < 1) splits = 1;
  // equal parts, so that each part's list is as deep into the row's alternatives as the others
  p.split_cols = splits > 1 ? ((vocab + splits - 1) / splits + 7) / 8 * 8 : vocab;
  p.splits = (int)((vocab + p.split_cols - 1) / p.split_cols);
  trips = (p.split_cols + trip - 1) / trip;
  const int64_t most = kGroupBytes / (int64_t)sizeof(unsigned) / p.threads;  // words per thread
  p.span = (int)((trips + most - 1) / most);
  p.slots = (trips + p.span - 1) / p.span * p.threads;
  return p;
}

template <class D, bool VEC, int NT>
void launch_topk(const TopkArgs& a, int64_t workgroups, size_t lds_bytes, hipStream_t s) {
  hipLaunchKernelGGL((row_topk_kernel<D, VEC, NT>), dim3((unsigned)workgroups), dim3(NT), lds_bytes, s, a);
}
template <class D, bool VEC>
void launch_divergence(const DivergenceArgs& a, int64_t n_rows, hipStream_t s) {
  // few long rows: row_softmax.hip's launch_stats()
  if (n_rows <= device_cu_count() && a.cols * (int64_t)sizeof(typename D::type) >= 64 * 1024)
    hipLaunchKernelGGL((row_divergence_kernel<D, VEC, kWide>), dim3((unsigned)n_rows), dim3(kWide), 0, s, a);
  else
    hipLaunchKernelGGL((row_divergence_kernel<D, VEC, kNarrow>), dim3((unsigned)n_rows), dim3(kNarrow), 0, s, a);
}

int check_topk(const char* what, const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t ld, int k,
               float rcp_temperature) {
  int st = check_rows(what, logits, dtype, n_rows, vocab, ld);
  if (st != VAMD_OK) return st;
  VAMD_REQUIRE(vocab < (1ll << 31), "%s: vocab too large", what);
  VAMD_REQUIRE(k >= 1 && k <= kMaxK, "%s: k is %d, of 1 to %d", what, k, kMaxK);
  VAMD_REQUIRE(rcp_temperature > 0.f && rcp_temperature < kInf, "%s: temperature must be positive", what);
  return VAMD_OK;
}

int chunk_columns(int dtype) {
  return kNarrow * (dtype == VAMD_DT_F32 ? F32::kVec * F32::kBackwardLoads : BF16::kVec * BF16::kBackwardLoads);
}
static_assert(BF16::kVec * BF16::kBackwardLoads == F16::kVec * F16::kBackwardLoads, "chunk_columns");
int64_t chunks_of(int64_t vocab, int dtype) { return (vocab + chunk_columns(dtype) - 1) / chunk_columns(dtype); }
// of the sorted entries, none where they are few
size_t sorted_bytes(int64_t n_rows, int64_t vocab, int dtype, int k) {
  if (k <= kUnsortedEntries) return 0;
  return 2 * align_up((size_t)n_rows * k * 4, 256) + align_up((size_t)n_rows * (chunks_of(vocab, dtype) + 1) * 4, 256);
}
Sorted carve_sorted(void* buffer, int64_t n_rows, int64_t vocab, int dtype, int k) {
  Sorted to{};
  if (k <= kUnsortedEntries || !buffer) return to;
  to.chunks = (int)chunks_of(vocab, dtype);
  to.chunk_cols = chunk_columns(dtype);
  Carver carve(buffer);
  to.column = carve.take<int>((size_t)n_rows * k);
  to.grad = carve.take<float>((size_t)n_rows * k);
  to.first = carve.take<int>((size_t)n_rows * (to.chunks + 1));
  return to;
}
size_t entries_bytes(int64_t n_rows, int64_t vocab, int dtype, int k) {
  const size_t many = sorted_bytes(n_rows, vocab, dtype, k);
  return many ? many : (size_t)n_rows * k * 4;
}
int check_backward(const char* what, const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t ld, int k,
                   float rcp_temperature, const float* stats, const void* d_logits, int64_t ld_out) {
  const int st = check_topk(what, logits, dtype, n_rows, vocab, ld, k, rcp_temperature);
  if (st != VAMD_OK) return st;
  VAMD_REQUIRE(stats && reinterpret_cast<uintptr_t>(stats) % 16 == 0, "%s: stats must be given, 16-byte aligned", what);
  VAMD_REQUIRE(d_logits && ld_out >= vocab && d_logits != logits, "%s: bad output", what);
  VAMD_REQUIRE(n_rows * chunks_of(vocab, dtype) < (1ll << 31), "%s: too many workgroups", what);
  return VAMD_OK;
}
template <class D, bool ENTROPY>
void launch_backward(const EntriesArgs& a, bool vec, bool stream, bool sorted, int64_t n_rows, hipStream_t s) {
  void (*const kernels[2][2][2])(EntriesArgs) = {
      {{row_entries_backward_kernel<D, false, false, false, ENTROPY>, row_entries_backward_kernel<D, false, false, true, ENTROPY>},
       {row_entries_backward_kernel<D, false, true, false, ENTROPY>, row_entries_backward_kernel<D, false, true, true, ENTROPY>}},
      {{row_entries_backward_kernel<D, true, false, false, ENTROPY>, row_entries_backward_kernel<D, true, false, true, ENTROPY>},
       {row_entries_backward_kernel<D, true, true, false, ENTROPY>, row_entries_backward_kernel<D, true, true, true, ENTROPY>}}};
  hipLaunchKernelGGL(kernels[vec][stream][sorted], dim3((unsigned)(n_rows * a.chunks)), dim3(kNarrow), 0, s, a);
}
int entries_backward(EntriesArgs a, int dtype, int64_t n_rows, hipStream_t s) {
  a.chunks = (int)chunks_of(a.cols, dtype);
  const bool sorted = a.sorted.column != nullptr;
  VAMD_DTYPE_DISPATCH(dtype, D, {
    const bool vec = rows_vectorizable<D>(a.logits, a.ld) && rows_vectorizable<D>(a.out, a.ld_out);
    const bool stream = cached_rows(n_rows, a.ld, sizeof(typename D::type)) < n_rows;
    const auto launch = a.d_entropy ? launch_backward<D, true> : launch_backward<D, false>;
    launch(a, vec, stream, sorted, n_rows, s);
  });
  VAMD_LAUNCH_CHECK();
  return VAMD_OK;
}

}  // namespace

int launch_head_pick(const HeadPickArgs& a, hipStream_t s) {
  const size_t list = kCandidates * sizeof(uint64_t), maxima = (size_t)a.groups * sizeof(float);
  if (threads_for(a.k) == kNarrow)
    hipLaunchKernelGGL((head_pick_kernel<kNarrow>), dim3((unsigned)a.n_tokens), dim3(kNarrow), maxima > list ? maxima : list, s, a);
  else
    hipLaunchKernelGGL((head_pick_kernel<kMiddle>), dim3((unsigned)a.n_tokens), dim3(kMiddle), maxima > list ? maxima : list, s, a);
  VAMD_LAUNCH_CHECK();
  return VAMD_OK;
}

}  // namespace vamd

using namespace vamd;

extern "C" size_t vamd_row_topk_workspace_bytes(int64_t n_rows, int64_t vocab, int dtype, int k) {
  if (n_rows <= 0 || vocab <= 0 || k <= 0 || k > kMaxK) return 0;
  const TopkPlan p = plan_topk(n_rows, vocab, dtype, k);
  if (p.splits == 1) return 0;
  const size_t parts = (size_t)n_rows * p.splits;
  return align_up(parts * sizeof(float4), 256) + align_up(parts * k * sizeof(uint64_t), 256);
}

extern "C" int vamd_row_topk(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t ld, const int64_t* labels,
                             int k, float rcp_temperature, float* logprobs, float* entropy, float* top, int64_t* index,
                             float* stats, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_topk("row_topk", logits, dtype, n_rows, vocab, ld, k, rcp_temperature);
  if (st != VAMD_OK) return st;
  VAMD_REQUIRE(k <= vocab, "row_topk: %d alternatives of %lld", k, (long long)vocab);
  VAMD_REQUIRE(top && index, "row_topk: null output");
  VAMD_REQUIRE(!logprobs || labels, "row_topk: logprobs need labels");
  VAMD_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 16 == 0, "row_topk: stats must be 16-byte aligned");
  const TopkPlan p = plan_topk(n_rows, vocab, dtype, k);
  const size_t need = vamd_row_topk_workspace_bytes(n_rows, vocab, dtype, k);
  if (need && (!workspace || workspace_bytes < need)) {
    set_error("row_topk: workspace %zu bytes, need %zu", workspace_bytes, need);
    return VAMD_EWORKSPACE;
  }
  VAMD_REQUIRE(n_rows * p.splits < (1ll << 31), "row_topk: too many workgroups");
  TopkArgs a{logits, ld, vocab, labels, k, p.span, rcp_temperature * kLog2e, rcp_temperature, logprobs, entropy, top, index,
             reinterpret_cast<float4*>(stats), 0, p.splits, p.split_cols, nullptr, nullptr};
  if (need) {
    Carver carve(workspace);
    a.part_state = carve.take<float4>((size_t)n_rows * p.splits);
    a.part_entry = carve.take<uint64_t>((size_t)n_rows * p.splits * k);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  VAMD_DTYPE_DISPATCH(dtype, D, {
    a.cached_rows = cached_rows(n_rows, ld, sizeof(typename D::type));
    const bool vec = rows_vectorizable<D>(logits, ld);
    const auto launch = p.threads == kNarrow ? (vec ? launch_topk<D, true, kNarrow> : launch_topk<D, false, kNarrow>)
                                             : (vec ? launch_topk<D, true, kMiddle> : launch_topk<D, false, kMiddle>);
    launch(a, n_rows * p.splits, p.lds_bytes(), s);
    if (p.splits > 1) {
      VAMD_LAUNCH_CHECK();
      hipLaunchKernelGGL((row_topk_join_kernel<D>), dim3((unsigned)n_rows), dim3(kNarrow),
                         kJoinEntries * sizeof(uint64_t), s, a);
    }
  });
  VAMD_LAUNCH_CHECK();
  return VAMD_OK;
}

extern "C" size_t vamd_row_topk_backward_workspace_bytes(int64_t n_rows, int64_t vocab, int dtype, int k) {
  if (n_rows <= 0 || vocab <= 0 || k <= 0 || k > kMaxK) return 0;
  return align_up((size_t)n_rows * 4, 256) + sorted_bytes(n_rows, vocab, dtype, k);
}

extern "C" int vamd_row_topk_backward(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t ld,
                                      const int64_t* labels, int k, const int64_t* index, float rcp_temperature,
                                      const float* stats, const float* d_logprobs, const float* d_entropy,
                                      const float* d_top, void* d_logits, int64_t ld_out, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  const int st = check_backward("row_topk_backward", logits, dtype, n_rows, vocab, ld, k, rcp_temperature, stats, d_logits, ld_out);
  if (st != VAMD_OK) return st;
  VAMD_REQUIRE(d_logprobs || d_entropy || d_top, "row_topk_backward: no upstream gradient");
  VAMD_REQUIRE((!d_logprobs || labels) && (!d_top || index), "row_topk_backward: gradients of log-probs need their tokens");
  const size_t need = vamd_row_topk_backward_workspace_bytes(n_rows, vocab, dtype, k);
  if (!workspace || workspace_bytes < need) {
    set_error("row_topk_backward: workspace %zu bytes, need %zu", workspace_bytes, need);
    return VAMD_EWORKSPACE;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* const weight = static_cast<float*>(workspace);
  const int entries = d_top ? k : 0;
  const Sorted sorted =
      carve_sorted(static_cast<char*>(workspace) + align_up((size_t)n_rows * 4, 256), n_rows, vocab, dtype, entries);
  hipLaunchKernelGGL(row_topk_prepare_kernel, dim3((unsigned)n_rows), dim3(kNarrow), 0, s, d_logprobs, labels, vocab, d_top, index,
                     entries, weight, sorted);
  VAMD_LAUNCH_CHECK();
  return entries_backward(EntriesArgs{logits, ld, vocab, 0, entries, index, d_top, sorted, reinterpret_cast<const float4*>(stats),
                                      weight, nullptr, labels, d_logprobs, d_entropy, rcp_temperature * kLog2e, rcp_temperature,
                                      d_logits, ld_out},
                          dtype, n_rows, s);
}

extern "C" size_t vamd_row_divergence_entries_bytes(int64_t n_rows, int64_t vocab, int dtype, int k) {
  if (n_rows <= 0 || vocab <= 0 || k <= 0 || k > kMaxK) return 0;
  return entries_bytes(n_rows, vocab, dtype, k);
}

extern "C" int vamd_row_divergence(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t ld,
                                   const float* teacher_logprobs, const int64_t* teacher_index, int k, int divergence,
                                   float beta, float rcp_temperature, float* loss, float* stats, void* entries,
                                   size_t entries_size, void* stream) {
  int st = check_topk("row_divergence", logits, dtype, n_rows, vocab, ld, k, rcp_temperature);
  if (st != VAMD_OK) return st;
  if ((st = check_divergence("row_divergence", k, divergence, beta)) != VAMD_OK) return st;
  VAMD_REQUIRE(teacher_logprobs && teacher_index && loss, "row_divergence: null pointer");
  VAMD_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 16 == 0, "row_divergence: stats must be 16-byte aligned");
  VAMD_REQUIRE((stats == nullptr) == (entries == nullptr), "row_divergence: stats and entries are written together or not at all");
  if (entries && entries_size < entries_bytes(n_rows, vocab, dtype, k)) {
    set_error("row_divergence: entries of %zu bytes, need %zu", entries_size, entries_bytes(n_rows, vocab, dtype, k));
    return VAMD_EWORKSPACE;
  }
  DivergenceArgs a{logits, ld, vocab, teacher_logprobs, teacher_index, k, divergence, beta, rcp_temperature * kLog2e, loss,
                   reinterpret_cast<float4*>(stats), k <= kUnsortedEntries ? static_cast<float*>(entries) : nullptr,
                   carve_sorted(entries, n_rows, vocab, dtype, k), 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  VAMD_DTYPE_DISPATCH(dtype, D, {
    a.cached_rows = cached_rows(n_rows, ld, sizeof(typename D::type));
    if (rows_vectorizable<D>(logits, ld)) launch_divergence<D, true>(a, n_rows, s);
    else launch_divergence<D, false>(a, n_rows, s);
  });
  VAMD_LAUNCH_CHECK();
  return VAMD_OK;
}

extern "C" int vamd_row_divergence_backward(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t ld,
                                            const int64_t* teacher_index, int k, float rcp_temperature, const float* stats,
                                            const void* entries, const float* d_loss, void* d_logits, int64_t ld_out,
                                            void* stream) {
  const int st = check_backward("row_divergence_backward", logits, dtype, n_rows, vocab, ld, k, rcp_temperature, stats, d_logits,
                                ld_out);
  if (st != VAMD_OK) return st;
  VAMD_REQUIRE(teacher_index && entries && d_loss, "row_divergence_backward: null pointer");
  return entries_backward(EntriesArgs{logits, ld, vocab, 0, k, teacher_index, static_cast<const float*>(entries),
                                      carve_sorted(const_cast<void*>(entries), n_rows, vocab, dtype, k),
                                      reinterpret_cast<const float4*>(stats), nullptr, d_loss, nullptr, nullptr, nullptr,
                                      rcp_temperature * kLog2e, rcp_temperature, d_logits, ld_out},
                          dtype, n_rows, static_cast<hipStream_t>(stream));
}
