// Categorical rows: log-probabilities of given categories with the row's entropy and its most probable alternatives, the
// gradient of those, and distillation from a teacher's top logits (loss and gradient).
//
// A row is n <= V logits x of one categorical entry.  With c = log2(e) / T, m = max x and d_v = c (x_v - m):
//   s = sum_v 2^d_v = 1 + r,   log q_v = ln2 d_v - log1p(r),   H = log1p(r) + ln2 u / s,   u = -sum_v 2^d_v d_v.
// r and u are sums over the categories OTHER than the largest one (its terms are 1 and 0 exactly), so a row that is
// nearly certain of one category keeps the relative accuracy of its log-probability and entropy: 1 + r would round r to
// 6e-8.  Partial results (of a thread, a workgroup, a part of a row) carry (m, s or r, u) and are joined by rescaling
// with 2^(c (m_part - m)).  All sums are held in 32 bits, the sum of the losses of all rows in 64.
#include "dmv_common.h"
#include "dmv_objmath.h"

#include <type_traits>

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kClampD = -256.f;        // 2^d (and e^d) is 0 below: keeps 0 * (-inf) out of sums and products
constexpr float kNearCertain = 0.0625f;  // below this r the largest category's thread sums its other terms again
constexpr int kMaxTop = DMV_CAT_MAX_TOP;
constexpr int kMaxTeacher = DMV_CAT_MAX_TEACHER;
constexpr int kMaxParts = 64;            // workgroups per row: a lane of the join each

// ------------------------------------------------------------------------------------------ elements
// 16 bytes of a row whose address is only element-aligned: one 16-byte access (the hardware takes any alignment)
struct __attribute__((packed, aligned(2))) Raw16 {
  uint32_t w[4];
};
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

template <int DT>
struct Elem;
template <>
struct Elem<DMV_F32> {
  typedef float type;
  static constexpr int N = 4;
  static constexpr int kOpenBits = 0;    // low bits of an order key that no two values of the type differ in alone
  static __device__ __forceinline__ float load(const void* p, int64_t i) { return ((const float*)p)[i]; }
  static __device__ __forceinline__ void store(void* p, int64_t i, float v) { ((float*)p)[i] = v; }
  static __device__ __forceinline__ void unpack(const Raw16& r, float* v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(r.w[e]);
  }
  static __device__ __forceinline__ void pack(const float* v, Raw16& r) {
#pragma unroll
    for (int e = 0; e < 4; ++e) r.w[e] = __float_as_uint(v[e]);
  }
};
template <>
struct Elem<DMV_BF16> {
  typedef uint16_t type;
  static constexpr int N = 8;
  static constexpr int kOpenBits = 16;
  static __device__ __forceinline__ float load(const void* p, int64_t i) {
    return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
  }
  static __device__ __forceinline__ void store(void* p, int64_t i, float v) { ((__bf16*)p)[i] = (__bf16)v; }
  static __device__ __forceinline__ void unpack(const Raw16& r, float* v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(r.w[e] << 16);
      v[2 * e + 1] = __uint_as_float(r.w[e] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void pack(const float* v, Raw16& r) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      r.w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){v[2 * e], v[2 * e + 1]}, bf16x2_t));
  }
};
template <>
struct Elem<DMV_F16> {
  typedef _Float16 type;
  static constexpr int N = 8;
  static constexpr int kOpenBits = 13;
  static __device__ __forceinline__ float load(const void* p, int64_t i) { return (float)((const _Float16*)p)[i]; }
  static __device__ __forceinline__ void store(void* p, int64_t i, float v) { ((_Float16*)p)[i] = (_Float16)v; }
  static __device__ __forceinline__ void unpack(const Raw16& r, float* v) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const h2 h = __builtin_bit_cast(h2, r.w[e]);
      v[2 * e] = (float)h[0];
      v[2 * e + 1] = (float)h[1];
    }
  }
  static __device__ __forceinline__ void pack(const float* v, Raw16& r) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; ++e) r.w[e] = __builtin_bit_cast(uint32_t, (h2){(_Float16)v[2 * e], (_Float16)v[2 * e + 1]});
  }
};
static inline int elem_size(int dt) { return dt == DMV_F32 ? 4 : 2; }
static inline int vec_elems(int dt) { return dt == DMV_F32 ? 4 : 8; }

// Order of the selection: larger values first, lower index first among equal ones (-0 and +0 are equal).  The key grows
// with the value; a 16-bit value's key is determined by its upper half.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kKeyMinusInf = 0x007fffffu;  // order_key(-inf)

// max(a, b, c) in one instruction; what is NaN is left out (fmaxf costs another instruction per operand whose origin the
// compiler does not know)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
template <int N>
__device__ __forceinline__ float max_of(const float* v, float m) {
  if constexpr (N == 1) return max3(v[0], m, m);
#pragma unroll
  for (int e = 0; e + 1 < N; e += 2) m = max3(v[e], v[e + 1], m);
  return m;
}

// log(1 + r), r >= 0 (or NaN), to a few ulp of itself: a series below 2^-6, else log u r / (u - 1) with u = fl(1 + r), in
// which the rounding of u cancels; the reciprocal unit's ulp is all that is added
__device__ __forceinline__ float log1p_row(float r) {
  const float u = 1.f + r;
  const float far = r < INFINITY ? __logf(u) * (r * __builtin_amdgcn_rcpf(u - 1.f)) : r;
  const float near = r * (1.f - r * (0.5f - r * (1.f / 3.f - r * (0.25f - r * 0.2f))));
  return r < 0x1p-6f ? near : far;
}

__device__ __forceinline__ float exp2_hw(float d) { return __builtin_amdgcn_exp2f(d); }

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_move_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
// v of the other 16 lanes of 32, or of the other 32 lanes: the exchange gives each lane both its own and the other's, in
// either order, which is all that a commutative operation needs
template <int X, typename Op>
__device__ __forceinline__ uint32_t across(uint32_t v, Op op) {
  if constexpr (X == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return op(r[0], r[1]);
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return op(r[0], r[1]);
  }
}
template <int R>
__device__ __forceinline__ uint32_t gmax_u(uint32_t v) {
  auto larger = [](uint32_t a, uint32_t b) { return max(a, b); };
  if (R >= 2) v = max(v, dpp_move_u<0xB1>(v));
  if (R >= 4) v = max(v, dpp_move_u<0x4E>(v));
  if (R >= 8) v = max(v, dpp_move_u<0x141>(v));
  if (R >= 16) v = max(v, dpp_move_u<0x140>(v));
  if (R >= 32) v = across<16>(v, larger);
  if (R >= 64) v = across<32>(v, larger);
  return v;
}
template <int R>
__device__ __forceinline__ uint32_t rsum_u(uint32_t v) {
  auto add = [](uint32_t a, uint32_t b) { return a + b; };
  if (R >= 2) v += dpp_move_u<0xB1>(v);
  if (R >= 4) v += dpp_move_u<0x4E>(v);
  if (R >= 8) v += dpp_move_u<0x141>(v);
  if (R >= 16) v += dpp_move_u<0x140>(v);
  if (R >= 32) v = across<16>(v, add);
  if (R >= 64) v = across<32>(v, add);
  return v;
}
template <int R>
__device__ __forceinline__ float rsum(float v) {
  auto add = [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); };
  if (R >= 2) v += dpp_move<0xB1>(v);
  if (R >= 4) v += dpp_move<0x4E>(v);
  if (R >= 8) v += dpp_move<0x141>(v);
  if (R >= 16) v += dpp_move<0x140>(v);
  if (R >= 32) v = __uint_as_float(across<16>(__float_as_uint(v), add));
  if (R >= 64) v = __uint_as_float(across<32>(__float_as_uint(v), add));
  return v;
}

// Largest of R lanes' values, as integers of the same order: a float maximum costs two more instructions a step (its
// operands' NaNs are quietened first), an integer one takes the lane exchange as an operand.
template <int R>
__device__ __forceinline__ float gmax(float v) {
  const int b = __float_as_int(v);
  int k = b ^ ((b >> 31) & 0x7fffffff);
  if (R >= 2) k = max(k, (int)dpp_move_u<0xB1>((uint32_t)k));
  if (R >= 4) k = max(k, (int)dpp_move_u<0x4E>((uint32_t)k));
  if (R >= 8) k = max(k, (int)dpp_move_u<0x141>((uint32_t)k));
  if (R >= 16) k = max(k, (int)dpp_move_u<0x140>((uint32_t)k));
  auto larger = [](uint32_t a, uint32_t b) { return (uint32_t)max((int)a, (int)b); };
  if (R >= 32) k = (int)across<16>((uint32_t)k, larger);
  if (R >= 64) k = (int)across<32>((uint32_t)k, larger);
  return __int_as_float(k ^ ((k >> 31) & 0x7fffffff));
}

// ------------------------------------------------------------------------------------------ arguments
struct Rows {
  const char* x;
  int64_t ld, rows;  // pitch in elements
  int V;
  const int64_t* X;
  const uint8_t* M;
  const int32_t* sizes;
  int64_t x_period, m_period, size_period;
};

// entry of a per-row array that repeats with `period` rows (there are fewer than 2^31 rows)
__device__ __forceinline__ int64_t wrap(int64_t row, int64_t period, int64_t rows) {
  return period >= rows ? row : (int64_t)((uint32_t)row % (uint32_t)period);
}
__device__ __forceinline__ int row_size(const Rows& a, int64_t row) {
  if (!a.sizes) return a.V;
  const int n = a.sizes[wrap(row, a.size_period, a.rows)];
  return n < 0 ? 0 : (n > a.V ? a.V : n);
}
__device__ __forceinline__ bool row_seen(const Rows& a, int64_t row) { return !a.M || a.M[wrap(row, a.m_period, a.rows)] != 0; }

struct Fwd {
  Rows r;
  float* log_prob;
  float* entropy;
  int top;
  float* top_lp;
  int64_t* top_idx;
  f32x4* stats;  // per row (m, 1 / s, log s, H): what the gradient reads; 1 / s = 0: nothing of non-zero probability
  float c;       // log2(e) / T
  int parts;     // workgroups per row; > 1: partial results go to ws
  f32x4* part;   // [rows][parts] (m, r, u, -)
  uint2* part_top;  // [rows][parts][top] (key, index), in order; key 0 past the end
  const float* weight;  // nullable, for distillation: rows of weight 0 are not read
  int64_t w_period;
};

struct Bwd {
  Rows r;
  const f32x4* stats;
  const float* g_lp;
  const float* g_ent;
  int top;
  const int64_t* top_idx;
  const float* g_top;
  void* d;
  int64_t ld_d;
  int chunks;
};

struct Teacher {
  const void* t;
  const int64_t* idx;
  const float* weight;
  int64_t t_period, w_period;
  int k, dt;
  float c;      // log2(e) / T
  float inv_T;
};

struct Dist {
  Rows r;
  Teacher t;
  float* per_row;
  double* loss_part;  // one per workgroup of the launch
  float* loss;        // the loss itself, if the launch has one workgroup
  f32x4* stats;
  const float* gscale;
  int unless_one;  // the gradient of gscale = 1 is already in place
  void* d;         // nullable: loss only
  int64_t ld_d;
  int chunks, parts;
  f32x4* part;
};

__device__ __forceinline__ float teacher_logit(const Teacher& t, int64_t i) {
  if (t.dt == DMV_F32) return Elem<DMV_F32>::load(t.t, i);
  if (t.dt == DMV_BF16) return Elem<DMV_BF16>::load(t.t, i);
  return Elem<DMV_F16>::load(t.t, i);
}

// Slot `s` of a row = its elements [s VEC, s VEC + VEC).  The access starts at min(s VEC, V - VEC), so it never leaves the
// row (V >= VEC): the last slot of a row whose length is no multiple of VEC overlaps the one before.
template <int VEC>
__device__ __forceinline__ int slot_base(int s, int V) {
  const int b = s * VEC;
  return b + VEC <= V ? b : V - VEC;
}
// Slots of a long row, cut where its addresses are multiples of 16: slot s = elements [s VEC - lead, s VEC - lead + VEC) below
// n.  Accesses stay inside the row as above; a first and a last slot overlap their neighbours.  (Cut at the row's start,
// rows of odd length take a fifth longer to read: 1024 x 50001 float16 27 us, x 50000 23 us.)
template <int VEC>
struct Span {
  int lead, V, n, slots;
  __device__ __forceinline__ Span(const char* p, int elem, int V_, int n_) : V(V_), n(n_) {
    lead = (int)(((uintptr_t)p & 15) / elem);
    slots = n > 0 ? (n + lead + VEC - 1) / VEC : 0;
  }
  __device__ __forceinline__ int base(int s) const {
    const int f = s * VEC - lead;
    return f < 0 ? 0 : (f + VEC <= V ? f : V - VEC);
  }
  __device__ __forceinline__ bool whole(int s) const { return s * VEC >= lead && s * VEC - lead + VEC <= n; }
  __device__ __forceinline__ bool holds(int s, int i) const {
    const int f = s * VEC - lead;
    return i >= f && i < f + VEC && i < n;
  }
};
template <int DT, int VEC>
__device__ __forceinline__ void slot_load(const char* row, int base, float* v) {
  if constexpr (VEC == 1) {
    v[0] = Elem<DT>::load(row, base);
  } else {
    static_assert(VEC == Elem<DT>::N, "");
    Elem<DT>::unpack(*(const Raw16*)(row + (int64_t)base * (int)sizeof(typename Elem<DT>::type)), v);
  }
}
template <int DT, int VEC>
__device__ __forceinline__ void slot_store(char* row, int base, const float* v) {
  if constexpr (VEC == 1) {
    Elem<DT>::store(row, base, v[0]);
  } else {
    Raw16 r;
    Elem<DT>::pack(v, r);
    *(Raw16*)(row + (int64_t)base * (int)sizeof(typename Elem<DT>::type)) = r;
  }
}

// ------------------------------------------------------------------------------------------ gradient of one row
// With S = g_lp + sum_j g_top[j] and a_v what of S belongs to category v itself:
//   dx_v = a_v - S q_v - g_H q_v (log q_v + H)
// The dense part (a_v = 0) is written for every category; the few with a_v != 0 are written again by `at`, with
// a_v (1 - q_v) as -a_v expm1(log q_v): no cancellation where q_v is close to 1.
struct RowGrad {
  float m, inv_s, logs, S, gh, H;
  __device__ __forceinline__ float dense(float x) const {
    const float y = x - m;
    const float q = exp2_hw(y * kLog2e) * inv_s;
    return -q * (S + gh * (fmaxf(y - logs, kClampD) + H));
  }
  __device__ __forceinline__ float at(float x, float a) const {
    const float lq = fmaxf(x - m - logs, kClampD);
    const float q = exp2_hw(lq * kLog2e);
    return -a * expm1f(lq) - (S - a) * q - gh * q * (lq + H);
  }
};

// ------------------------------------------------------------------------------------------ short rows
// L lanes hold a row of up to 32 L elements in registers (SL slots of VEC elements each); 64 / L rows per wavefront.  What a
// row costs apart from its elements (addresses, reductions, logarithm, outputs) is as much for 4 lanes as for 64, so L is
// the smallest that holds the row.
constexpr int kSmallThreads = 256;
constexpr int kSmallMax = DMV_CAT_SHORT_ROW;   // their longest row: 64 lanes, 32 elements each

// Candidates of a selection: key in the upper half, ~index in the lower, so that the larger number is the better one.
typedef unsigned long long cand_t;
__device__ __forceinline__ cand_t candidate(uint32_t key, uint32_t index) { return ((cand_t)key << 32) | (uint32_t)~index; }

// The values of a packed slot for one pass over the row.  The compiler is made to forget what it knows of them and to keep
// the slots in order: it would otherwise hold the unpacked values, twice the registers, across the passes.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <int DT>
__device__ __forceinline__ void pass_over(u32x4& r, float* v) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" : "+v"(r));
  Elem<DT>::unpack(__builtin_bit_cast(Raw16, r), v);
}
__device__ __forceinline__ int again(int t) {
  asm volatile("" : "+v"(t));
  return t;
}

template <int DT, int VEC>
struct SmallSlot {
  u32x4 raw;
  __device__ __forceinline__ void load(const char* p, int base) {
    raw = __builtin_bit_cast(u32x4, *(const Raw16*)(p + (int64_t)base * (int)sizeof(typename Elem<DT>::type)));
  }
  __device__ __forceinline__ void unpack(float* v) const { Elem<DT>::unpack(__builtin_bit_cast(Raw16, raw), v); }
  __device__ __forceinline__ void pass(float* v) { pass_over<DT>(raw, v); }
  __device__ __forceinline__ void pack(const float* v) {
    Raw16 r;
    Elem<DT>::pack(v, r);
    raw = __builtin_bit_cast(u32x4, r);
  }
};
template <int DT>
struct SmallSlot<DT, 1> {
  float x;
  __device__ __forceinline__ void load(const char* p, int base) { x = Elem<DT>::load(p, base); }
  __device__ __forceinline__ void unpack(float* v) const { v[0] = x; }
  __device__ __forceinline__ void pass(float* v) { v[0] = x; }
  __device__ __forceinline__ void pack(const float* v) { x = v[0]; }
};

template <int DT, int VEC, int L, int SL>
struct SmallRow {
  static constexpr int E = VEC * SL;
  SmallSlot<DT, VEC> slot[SL];
  // (a lane without a slot gets the row's last one)
  __device__ __forceinline__ void load(const char* p, int V, int lane) {
#pragma unroll
    for (int j = 0; j < SL; ++j) {
      const int b = (lane + L * j) * VEC;
      slot[j].load(p, b + VEC <= V ? b : V - VEC);
    }
  }
  // every category once: what is past n, past the row, or shared with the slot before becomes -inf
  __device__ __forceinline__ void count_once(int V, int n, int lane) {
#pragma unroll
    for (int j = 0; j < SL; ++j) {
      const int f = (lane + L * j) * VEC;
      if (f + VEC > n) {
        const int b = f + VEC <= V ? f : V - VEC;
        float v[VEC];
        slot[j].unpack(v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = (b + e >= f && b + e < n) ? v[e] : -INFINITY;
        slot[j].pack(v);
      }
    }
  }
  __device__ __forceinline__ void values(float* o) const {
#pragma unroll
    for (int j = 0; j < SL; ++j) slot[j].unpack(o + j * VEC);
  }
};

// (m, r, u) of a row held by L lanes; r < 0: no category of non-zero probability.  The largest element's term is 1 and all
// others' are below (or round to 1, and count as such): the fractions sum to those of the others, and what the whole sum
// has more is the number of ones.  The row stays packed between the passes: unpacked it would take twice the registers,
// and the kernel half of its wavefronts.
// KEEP: the terms 2^(c (x - m)) go to `kept`.
template <bool ENT, bool KEEP, int DT, int VEC, int L, int SL>
__device__ __forceinline__ void small_stats(SmallRow<DT, VEC, L, SL>& x, float c, float& m, float& r, float& u, float* kept = nullptr) {
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < SL; ++j) {
    float v[VEC];
    x.slot[j].pass(v);
    mx = max_of<VEC>(v, mx);
  }
  m = gmax<L>(mx);
  const float ref = m == -INFINITY ? 0.f : m;
  float s = 0.f, f = 0.f, t = 0.f;
#pragma unroll
  for (int j = 0; j < SL; ++j) {
    float v[VEC];
    x.slot[j].pass(v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float d = (v[e] - ref) * c, w = exp2_hw(d);
      s += w;
      f += __builtin_amdgcn_fractf(w);
      if (ENT) t = fmaf(w, fmaxf(d, kClampD), t);
      if (KEEP) kept[j * VEC + e] = w;
    }
  }
  u = ENT ? -rsum<L>(t) : 0.f;
  const float others = rsum<L>(f);
  r = others + (rintf(rsum<L>(s) - others) - 1.f);
}

// The k largest of a row held by L lanes, through emit(rank, value, index) by any lane; index -1 past the finite values.
//
// The k-th largest of the largest values of NB parts of every lane's elements is a lower bound of the k-th largest element.
// With twice as many parts that hold elements as k, about 1.4 k elements reach it (the median of the parts' largest
// values): those go to the group's list in LDS and are ranked by counting.  A row may fill a quarter of its tile only, so
// the number of parts follows from what it fills; beyond 8 a lane the elements themselves are searched.  (10000 x 1092
// float16, 64 alternatives: 35 us a call; 520 by two parts a lane, whose bound more elements reach than the list holds.)
// When the list is too short all the same (many equal values): one rank at a time.
constexpr int kSmallList = 8;            // list entries per lane
// lanes of one wavefront that read what others of it wrote: in order without a wait
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
constexpr int kPops = 16;               // up to here the bound is found by taking the largest value k times
template <int NB, int E, int L>
__device__ __forceinline__ float small_bound(const float* o, int k) {
  constexpr int B = NB < E ? NB : E;          // (a tile of few elements has no more parts than those)
  float mx[B];
#pragma unroll
  for (int b = 0; b < B; ++b)
    if constexpr (E == B) mx[b] = o[b];
    else mx[b] = max_of<E / B>(o + b * (E / B), -INFINITY);
  if (B > 8 || k > kPops) {
    // the bound's bits one by one, below the exponent of the largest value if k values share it, until not many more than
    // k reach it (a key past that of +inf is a NaN's, which none reaches)
    const float first = max_of<B>(mx, -INFINITY);
    auto reach = [&](uint32_t t) {
      const float at = key_value(t);
      uint32_t c = 0;
#pragma unroll
      for (int b = 0; b < B; ++b) c += mx[b] >= at ? 1u : 0u;
      return (int)rsum_u<L>(c);
    };
    const uint32_t start = order_key(gmax<L>(first)) & 0xff800000u;
    int c = reach(start);
    const bool near = c >= k;
    uint32_t tau = near ? start : 0u;
    const int enough = k + (k >> 2) + 1;
    for (int bit = near ? 22 : 31; bit >= 0 && !(tau != 0u && c <= enough); --bit) {
      const uint32_t t = tau | (1u << bit);
      const int ct = reach(t);
      if (ct >= k) tau = t, c = ct;
    }
    return tau <= kKeyMinusInf ? -3.402823466e38f : fmaxf(key_value(tau), -3.402823466e38f);
  }
#pragma unroll
  for (int i = 1; i < B; ++i)                 // in order, largest first
#pragma unroll
    for (int j = i; j > 0; --j) {
      const float hi = max3(mx[j - 1], mx[j], mx[j]), lo = fminf(mx[j - 1], mx[j]);
      mx[j - 1] = hi, mx[j] = lo;
    }
  float bound;
  for (int t = k;;) {
    bound = gmax<L>(mx[0]);
    if (--t == 0) break;
    const bool mine = mx[0] == bound;
#pragma unroll
    for (int b = 0; b + 1 < B; ++b) mx[b] = mine ? mx[b + 1] : mx[b];
    mx[B - 1] = mine ? -INFINITY : mx[B - 1];
  }
  return fmaxf(bound, -3.402823466e38f);      // -inf is no alternative
}
template <int DT, int VEC, int L, int SL, typename Emit>
__device__ __forceinline__ void small_top(const float* o, const char* p, int V, int n, int lane, int k, cand_t* list, int* count,
                                          Emit emit) {
  constexpr int E = VEC * SL;
  static_assert(E <= 32, "");
  auto index = [&](int j, int e) { return slot_base<VEC>(lane + L * j, V) + e; };
  {
    // (tiles whose elements fit the list take the same number for all rows: rows of several sizes share a wavefront)
    const int filled = E <= kSmallList ? SL * L : (n + VEC - 1) / VEC, wanted = 2 * k * SL;
    const float bound = 2 * filled >= wanted   ? small_bound<2, E, L>(o, k)
                        : 4 * filled >= wanted ? small_bound<4, E, L>(o, k)
                        : 8 * filled >= wanted ? small_bound<8, E, L>(o, k)
                                               : small_bound<32, E, L>(o, k);
    uint32_t bits = 0;
#pragma unroll
    for (int i = E - 1; i >= 0; --i) bits = bits + bits + (o[i] >= bound ? 1u : 0u);
    if (lane == 0) *count = 0;
    wave_sync();
    if (bits) {
      int at = atomicAdd(count, __popc(bits));
      do {
        const int i = __ffs(bits) - 1;
        bits &= bits - 1;
        if (at < kSmallList * L) list[at] = (cand_t)(lane << 5 | i);
        ++at;
      } while (bits);
    }
    wave_sync();
    const int have = *count;
    if (have <= kSmallList * L) {
      for (int q = lane; q < have; q += L) {      // (their values are read again rather than picked from registers)
        const int id = (int)list[q], i = id & 31, at = slot_base<VEC>((id >> 5) + L * (i / VEC), V) + i % VEC;
        list[q] = candidate(order_key(Elem<DT>::load(p, at)), (uint32_t)at);
      }
      wave_sync();
      for (int i = lane; i < have; i += L) {
        const cand_t me = list[i];
        int rank = 0;
        for (int j = 0; j < have; ++j) rank += list[j] > me ? 1 : 0;
        if (rank < k) emit(rank, key_value((uint32_t)(me >> 32)), (int)~(uint32_t)me);
      }
      for (int j = have + lane; j < k; j += L) emit(j, -INFINITY, -1);
      return;
    }
  }
  // one rank at a time: what has been ranked is all that is better than the last one
  float last = INFINITY;
  int last_at = -1;
  for (int t = 0; t < k; ++t) {
    float best = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < SL; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float x = o[j * VEC + e];
        if ((x < last || (x == last && index(j, e) > last_at)) && x > best) {
          best = x;
          at = index(j, e);
        }
      }
    const float top = gmax<L>(best);
    const uint32_t low = ~gmax_u<L>(best == top ? ~(uint32_t)at : 0u);   // lowest index among the equal ones
    const bool none = top == -INFINITY;
    if (lane == (t & (L - 1))) emit(t, top, none ? -1 : (int)low);
    last = top;
    last_at = (int)low;
  }
}

// All of a row's elements in order, for k beyond the bound's reach (k > 4 L): a bitonic network over the E L elements, pairs
// within a lane or between lanes one or more apart.  Keys as candidate(); 16-bit types put their 16-bit key and the index
// into 32 bits, which halves the exchanges (and a comparison costs two instructions instead of five).
template <int DT>
struct SortKey {
  typedef uint32_t type;
  static __device__ __forceinline__ type of(float x, int i) {
    uint32_t k;
    if constexpr (DT == DMV_BF16) {
      k = order_key(x) >> 16;
    } else {
      const uint32_t b = __builtin_bit_cast(uint16_t, (_Float16)(x + 0.f));
      k = b & 0x8000u ? ~b & 0xffffu : b | 0x8000u;
    }
    return x > -INFINITY ? k << 16 | (~(uint32_t)i & 0xffffu) : 0u;
  }
  static __device__ __forceinline__ int index(type k) { return (int)(~k & 0xffffu); }
  static __device__ __forceinline__ float value(type k) {
    const uint32_t h = k >> 16;
    if constexpr (DT == DMV_BF16) return key_value(h & 0x8000u ? h << 16 : h << 16 | 0xffffu);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(h & 0x8000u ? h & 0x7fffu : ~h));
  }
};
template <>
struct SortKey<DMV_F32> {
  typedef cand_t type;
  static __device__ __forceinline__ type of(float x, int i) { return x > -INFINITY ? candidate(order_key(x), (uint32_t)i) : 0ull; }
  static __device__ __forceinline__ int index(type k) { return (int)~(uint32_t)k; }
  static __device__ __forceinline__ float value(type k) { return key_value((uint32_t)(k >> 32)); }
};
// the key of lane ^ X, X = 1, 2 or 4
template <int X>
__device__ __forceinline__ uint32_t lane_xor(uint32_t k) {
  if (X == 1) return dpp_move_u<0xB1>(k);
  if (X == 2) return dpp_move_u<0x4E>(k);
  return dpp_move_u<0x141>(dpp_move_u<0x1B>(k));        // 7 - (3 - lane within a quad): lane ^ 4
}
template <int X>
__device__ __forceinline__ cand_t lane_xor(cand_t k) {
  return (cand_t)lane_xor<X>((uint32_t)(k >> 32)) << 32 | lane_xor<X>((uint32_t)k);
}
template <int E, int SIZE, int STRIDE, typename K>
__device__ __forceinline__ void sort_stage(K* key, int lane) {
  // element lane E + e, largest first: a pair (i, i ^ STRIDE) is in descending order where i & SIZE is 0
  if constexpr (STRIDE >= E) {
    const bool low = (lane & (STRIDE / E)) == 0, down = (lane * E & SIZE) == 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const K other = lane_xor<STRIDE / E>(key[e]);
      key[e] = ((low == down) == (other > key[e])) ? other : key[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if ((e & STRIDE) == 0) {
        const bool down = SIZE < E ? (e & SIZE) == 0 : (lane * E & SIZE) == 0;
        const K a = key[e], b = key[e | STRIDE];
        const bool swap = (b > a) == down;
        key[e] = swap ? b : a;
        key[e | STRIDE] = swap ? a : b;
      }
  }
  if constexpr (STRIDE > 1) sort_stage<E, SIZE, STRIDE / 2>(key, lane);
}
template <int E, int L, int SIZE, typename K>
__device__ __forceinline__ void sort_down(K* key, int lane) {
  if constexpr (SIZE > 2) sort_down<E, L, SIZE / 2>(key, lane);
  sort_stage<E, SIZE, SIZE / 2>(key, lane);
}
template <int DT, int VEC, int L, int SL, typename Emit>
__device__ __forceinline__ void small_sorted(const float* o, int V, int lane, int k, Emit emit) {
  constexpr int E = VEC * SL;
  typename SortKey<DT>::type key[E];
#pragma unroll
  for (int j = 0; j < SL; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) key[j * VEC + e] = SortKey<DT>::of(o[j * VEC + e], slot_base<VEC>(lane + L * j, V) + e);
  sort_down<E, L, E * L>(key, lane);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int rank = lane * E + e;
    if (rank < k) emit(rank, SortKey<DT>::value(key[e]), key[e] ? SortKey<DT>::index(key[e]) : -1);
  }
  for (int j = E * L + lane; j < k; j += L) emit(j, -INFINITY, -1);
}

// Short rows, forward.  Bound by the vector units (92 % busy) and not by memory: of 743 instructions that a wavefront takes for
// eight rows of 256 bfloat16 with entropy and 4 alternatives, about half are the passes over the elements (unpack,
// maximum, exponential, two sums).  100352 such rows: 20.4 us (2.8 TB/s); without alternatives and entropy 13 us (4.0 TB/s);
// 200000 x 100 float32 14.4 us (5.5 TB/s).
enum { kNoTop = 0, kRanked = 1, kSorted = 2 };
template <int DT, int VEC, int L, int SL, bool ENT, int TOP>
__global__ void __launch_bounds__(kSmallThreads) k_cat_fwd_small(Fwd a) {
  constexpr int E = VEC * SL, NG = kSmallThreads / L, ES = sizeof(typename Elem<DT>::type);
  __shared__ cand_t lists[TOP == kRanked ? NG : 1][TOP == kRanked ? kSmallList * L : 1];
  __shared__ int counts[NG];
  const int lane = threadIdx.x & (L - 1), V = a.r.V;
  const int row = blockIdx.x * NG + threadIdx.x / L;          // (rows * 16 bytes fit 32 bits)
  if (row >= (int)a.r.rows) return;
  const bool seen = row_seen(a.r, row);
  if (!TOP && !ENT && !seen) {
    if (lane == 0) a.log_prob[(uint32_t)row] = 0.f;
    return;
  }
  const int n = row_size(a.r, row);
  const char* p = a.r.x + row * a.r.ld * ES;
  SmallRow<DT, VEC, L, SL> x;
  x.load(p, V, lane);
  bool given = false;
  float xX = 0.f;
  if (a.log_prob && seen) {
    const int64_t X = a.r.X[wrap(row, a.r.x_period, a.r.rows)];
    given = X >= 0 && X < n;
    if (given) xX = Elem<DT>::load(p, X);
  }
  float m, r, u;
  x.count_once(V, n, lane);
  small_stats<ENT, false>(x, a.c, m, r, u);
  const bool empty = m == -INFINITY && !(r != r);
  const float logs = empty ? 0.f : log1p_row(r), inv_s = empty ? 0.f : __builtin_amdgcn_rcpf(1.f + r);
  const float H = empty ? 0.f : fmaf(kLn2 * u, inv_s, logs);
  if (lane == 0) {
    if (a.log_prob) a.log_prob[(uint32_t)row] = !seen ? 0.f : (empty ? -INFINITY : (!given ? NAN : (xX - m) - logs));
    if (ENT) a.entropy[(uint32_t)row] = H;
    if (a.stats) a.stats[(uint32_t)row] = f32x4{m, inv_s, logs, H};
  }
  if constexpr (TOP != kNoTop) {
    float* lp = a.top_lp + (int64_t)row * a.top;
    int64_t* idx = a.top_idx + (int64_t)row * a.top;
    if (logs != logs) {
      for (int j = lane; j < a.top; j += L) lp[j] = NAN, idx[j] = -1;
    } else {
      auto emit = [&](int rank, float v, int i) {
        idx[rank] = i;
        lp[rank] = i < 0 ? -INFINITY : (v - m) - logs;
      };
      const int g = threadIdx.x / L;
      float o[E];
      x.values(o);
      if constexpr (TOP == kSorted) small_sorted<DT, VEC, L, SL>(o, V, lane, a.top, emit);
      else small_top<DT, VEC, L, SL>(o, p, V, n, lane, a.top, lists[TOP == kRanked ? g : 0], &counts[g], emit);
    }
  }
}

// a_v of the gradient's sparse part for category v: what of the given category and the top alternatives falls on it
__device__ __forceinline__ float own_share(const Bwd& a, int64_t row, int64_t v, int64_t X, float gl) {
  float s = v == X ? gl : 0.f;
  if (a.g_top)
    for (int j = 0; j < a.top; ++j)
      if (a.top_idx[row * a.top + j] == v) s += a.g_top[row * a.top + j];
  return s;
}

// S of a row (and its given category, -1 if none), the same in every lane of the R lanes that ask
template <int R>
__device__ __forceinline__ RowGrad row_grad(const Bwd& a, int64_t row, int lane, int n, int64_t& X, float& gl) {
  RowGrad g;
  X = -1;
  gl = 0.f;
  if (a.g_lp && row_seen(a.r, row)) {
    X = a.r.X[wrap(row, a.r.x_period, a.r.rows)];
    gl = a.g_lp[row];
    if (X < 0 || X >= n) gl = NAN;      // as the log-probability of no category at all
  }
  g.S = gl;
  if (a.g_top) {
    float s = 0.f;
    for (int j = lane; j < a.top; j += R)
      if (a.top_idx[row * a.top + j] >= 0) s += a.g_top[row * a.top + j];
    g.S += rsum<R>(s);
  }
  g.gh = a.g_ent ? a.g_ent[row] : 0.f;
  g.m = g.inv_s = g.logs = g.H = 0.f;
  if (g.S != 0.f || g.gh != 0.f || a.g_top) {
    const f32x4 st = a.stats[row];
    g.m = st[0], g.inv_s = st[1], g.logs = st[2], g.H = st[3];
  }
  return g;
}

template <int DT, int VEC, int L, int SL>
__global__ void __launch_bounds__(kSmallThreads) k_cat_bwd_small(Bwd a) {
  constexpr int ES = sizeof(typename Elem<DT>::type);
  const int lane = threadIdx.x & (L - 1);
  const int64_t row = (int64_t)blockIdx.x * (kSmallThreads / L) + threadIdx.x / L;
  if (row >= a.r.rows) return;
  const int n = row_size(a.r, row), V = a.r.V;
  int64_t X;
  float gl;
  const RowGrad g = row_grad<L>(a, row, lane, n, X, gl);
  const char* p = a.r.x + row * a.r.ld * ES;
  char* out = (char*)a.d + row * a.ld_d * ES;
  const bool live = (g.S != 0.f || g.gh != 0.f || a.g_top) && g.inv_s != 0.f;
  SmallRow<DT, VEC, L, SL> x;
  if (live) x.load(p, V, lane);
#pragma unroll
  for (int j = 0; j < SL; ++j) {
    const int s = lane + L * j;
    if (s * VEC >= V) continue;
    const int b = slot_base<VEC>(s, V);
    float o[VEC];
    if (live) {
      float v[VEC];
      x.slot[j].unpack(v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = b + e < n ? g.dense(v[e]) : 0.f;
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = 0.f;
    }
    slot_store<DT, VEC>(out, b, o);
  }
  if (!live) return;
  // the dense part before the few categories written again: stores of one wavefront stay in order
  wave_sync();
  const int entries = 1 + (a.g_top ? a.top : 0);
  for (int j = lane; j < entries; j += L) {
    const int64_t v = j == 0 ? X : a.top_idx[row * a.top + j - 1];
    if (v < 0 || v >= n) continue;
    Elem<DT>::store(out, v, g.at(Elem<DT>::load(p, v), own_share(a, row, v, X, gl)));
  }
}

// ------------------------------------------------------------------------------------------ distillation, shared parts
// Teacher entry j counts if its index is not negative and its logit not -inf; the counted ones are normalised among
// themselves.  An index past the row's categories, or a logit that is NaN or +inf, makes the row's loss NaN, and its gradient
// at all of the row's categories; past those a gradient is 0 whatever the row holds.
__device__ __forceinline__ bool entry_counts(float t, int64_t i) { return i >= 0 && t != -INFINITY; }

__device__ __forceinline__ float exp_hw(float x) { return exp2_hw(x * kLog2e); }
// q - p of their logarithms without its cancellation: p expm1(log q - log p), a series where that is small
__device__ __forceinline__ float q_minus_p(float lq, float lp) {
  const float x = lq - lp, p = exp_hw(lp);
  if (fabsf(x) < 0.35f)      // (the next term is below 2e-8 of the sum)
    return p * (x * (1.f + x * (1.f / 2 + x * (1.f / 6 + x * (1.f / 24 + x * (1.f / 120 + x * (1.f / 720 + x * (1.f / 5040))))))));
  return x < 1.f ? p * (exp_hw(x) - 1.f) : exp_hw(lq) - p;
}

// A teacher's entry in LDS: its logit, then log p; the student's logit, then log q of its category; category (-1: empty).
struct Entry {
  float t, x;
  int i;
};
constexpr int kFewEntries = 16;       // up to here a category given twice is looked for entry by entry
constexpr int kLoneThreads = 1024;    // the workgroup of a small launch, which also forms the loss: a second launch saved

template <int DT, int VEC, int L>
__device__ __forceinline__ void small_zeros(char* out, int V, int lane) {
  const float z[VEC] = {};
  for (int s = lane; s * VEC < V; s += L) slot_store<DT, VEC>(out, slot_base<VEC>(s, V), z);
}

template <int DT, int VEC, int L, int SL, int NT>
__global__ void __launch_bounds__(NT) k_cat_distill_small(Dist a) {
  // (the smallest tiles have fewer categories than a word has bits)
  constexpr int E = VEC * SL, ES = sizeof(typename Elem<DT>::type), WORDS = (E * L + 31) / 32, NG = NT / L;
  static_assert(WORDS >= 1 && WORDS * 32 >= E * L, "a bit for every category of the tile");
  constexpr bool LONE = NT == kLoneThreads;
  __shared__ double sums[NT / 64];
  __shared__ uint32_t given[NG][WORDS];
  extern __shared__ Entry entries[];    // [NG][k]
  const float gs = a.gscale ? *a.gscale : 1.f;
  if (a.unless_one && gs == 1.f) return;
  const int lane = threadIdx.x & (L - 1), V = a.r.V, K = a.t.k, g = threadIdx.x / L;
  double part = 0.0;
  for (int row = blockIdx.x * NG + g; row < (int)a.r.rows; row += NG) {
    const float w = a.t.weight ? a.t.weight[wrap(row, a.t.w_period, a.r.rows)] : 1.f;
    float kl = 0.f;
    if (w != 0.f) {
      const char* p = a.r.x + row * a.r.ld * ES;
      SmallRow<DT, VEC, L, SL> x;
      x.load(p, V, lane);
      const int n = row_size(a.r, row);
      Entry* own = entries + g * K;
      const int64_t t0 = wrap(row, a.t.t_period, a.r.rows) * K;
      float tm = -INFINITY;
      uint32_t flags = 0;                 // 1: an entry counts, 2: one that cannot be
      for (int j = lane; j < K; j += L) {
        const int64_t i = a.t.idx[t0 + j];
        const float t = teacher_logit(a.t, t0 + j);
        const bool counts = entry_counts(t, i), bad = counts && (i >= n || !(t < INFINITY));
        flags |= (counts ? 1u : 0u) | (bad ? 2u : 0u);
        if (counts) tm = fmaxf(tm, t);
        own[j] = Entry{t, counts && !bad ? Elem<DT>::load(p, i) : 0.f, counts && !bad ? (int)i : -1};
      }
      tm = gmax<L>(tm);
      flags = gmax_u<L>(flags);
      const bool any = flags != 0u, bad = flags >= 2u;
      float m, r, u, kept[E];
      x.count_once(V, n, lane);
      small_stats<false, true>(x, a.t.c, m, r, u, kept);      // (twice the registers of the packed row, but no second exp2)
      const bool empty = m == -INFINITY && !(r != r);
      const float logs = empty ? 0.f : log1p_row(r), inv_s = empty ? 0.f : __builtin_amdgcn_rcpf(1.f + r);
      const bool live = any && (!empty || bad);
      if (live && !bad) {
        float s = 0.f, held = 0.f;
        for (int j = lane; j < K; j += L)
          if (own[j].i >= 0) {
            if (own[j].t == tm) held += 1.f;
            else s += exp2_hw((own[j].t - tm) * a.t.c);
          }
        const float t_logs = log1p_row(rsum<L>(s) + (rsum<L>(held) - 1.f));
        for (int j = lane; j < K; j += L)
          if (own[j].i >= 0) {
            const float lp = (own[j].t - tm) * a.t.inv_T - t_logs, q = exp_hw(lp), lq = (own[j].x - m) * a.t.inv_T - logs;
            if (q > 0.f) kl += q * (lp - lq);
            own[j].t = lp;
            own[j].x = lq;
          }
        kl = rsum<L>(kl);
      }
      if (any && empty) kl = INFINITY;
      if (bad) kl = NAN;
      if (lane == 0) part += (double)w * (double)kl;
      if (a.d) {
        char* out = (char*)a.d + row * a.ld_d * ES;
        const float scale = bad ? NAN : gs * w * a.t.inv_T, f = scale * inv_s;
        if (!live) small_zeros<DT, VEC, L>(out, V, lane);
  #pragma unroll
        for (int j = 0; j < SL; ++j) {
          const int fst = (lane + L * j) * VEC;
          if (fst >= V || !live) continue;
          float v[VEC];
  #pragma unroll
          for (int e = 0; e < VEC; ++e) v[e] = f * kept[j * VEC + e];     // (what does not count: 0, or NaN)
          if (fst + VEC <= V) slot_store<DT, VEC>(out, fst, v);
          else {
  #pragma unroll
            for (int e = 0; e < VEC; ++e)
              if (V - VEC + e >= fst) Elem<DT>::store(out, V - VEC + e, v[e]);
          }
        }
        if (live && !(fabsf(f) < INFINITY)) {       // past the row's size 0 all the same
          wave_sync();
          for (int i = n + lane; i < V; i += L) Elem<DT>::store(out, i, 0.f);
        }
        if (live && !bad) {
          // A category given more than once has all its entries' probability in each of them.  Whether there is one is told
          // by a bit per category.
          bool twice = K <= kFewEntries;
          if (!twice) {
            for (int q = lane; q < WORDS; q += L) given[g][q] = 0u;
            wave_sync();
            for (int j = lane; j < K; j += L)
              if (own[j].i >= 0) {
                const uint32_t bit = 1u << (own[j].i & 31);
                twice = twice || (atomicOr(&given[g][own[j].i >> 5], bit) & bit) != 0u;
              }
            twice = gmax_u<L>(twice ? 1u : 0u) != 0u;
          }
          // the dense part before the teacher's categories are written again: stores of one wavefront stay in order
          wave_sync();
          for (int j = lane; j < K; j += L) {
            const Entry e = own[j];
            if (e.i < 0) continue;
            float lp = e.t;
            if (twice) {
              int same = 0;
              float sum = 0.f;
              for (int h = 0; h < K; ++h)
                if (own[h].i == e.i) sum += exp_hw(own[h].t), ++same;
              if (same > 1) lp = logf(sum);
            }
            Elem<DT>::store(out, e.i, scale * q_minus_p(e.x, lp));
          }
        }
      }
    } else if (a.d) {
      small_zeros<DT, VEC, L>((char*)a.d + row * a.ld_d * ES, V, lane);
    }
    if (lane == 0 && a.per_row) a.per_row[(uint32_t)row] = kl;
    if (!LONE) break;
  }
  // the workgroup's share of the loss, in a fixed order
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) part += __shfl_xor(part, off);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = part;
  __syncthreads();
  if (threadIdx.x == 0 && (LONE ? a.loss != nullptr : a.loss_part != nullptr)) {
    double s = 0.0;
    for (int i = 0; i < NT / 64; ++i) s += sums[i];
    if (LONE) *a.loss = (float)s;
    else a.loss_part[blockIdx.x] = s;
  }
}

// ------------------------------------------------------------------------------------------ long rows
template <int NT>
struct BlockRed {
  float x[3][NT / 64];
};
template <int NT>
__device__ __forceinline__ float block_max(float v, BlockRed<NT>& s) {
  v = gmax<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.x[0][threadIdx.x >> 6] = v;
  __syncthreads();
  float m = s.x[0][0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) m = fmaxf(m, s.x[0][i]);
  return m;
}
template <int NT>
__device__ __forceinline__ void block_sum3(float& p, float& q, float& w, BlockRed<NT>& s) {
  p = rsum<64>(p), q = rsum<64>(q), w = rsum<64>(w);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    s.x[0][threadIdx.x >> 6] = p;
    s.x[1][threadIdx.x >> 6] = q;
    s.x[2][threadIdx.x >> 6] = w;
  }
  __syncthreads();
  p = q = w = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) p += s.x[0][i], q += s.x[1][i], w += s.x[2][i];
}

// running (max, sum, entropy sum) of one thread
struct Online {
  float m = -INFINITY, s = 0.f, t = 0.f;
  // N values, the largest of them mx
  template <int N, bool ENT>
  __device__ __forceinline__ void add(const float* v, float mx, float c) {
    const float mn = max3(mx, m, m);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float shift = fmaxf((m - ref) * c, kClampD), f = exp2_hw(shift);
    if (ENT) t = f * fmaf(s, shift, t);
    s *= f;
    m = mn;
    float s1 = 0.f, t1 = 0.f;
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float d0 = (v[e] - ref) * c, w0 = exp2_hw(d0);
      const float d1 = (v[e + 1] - ref) * c, w1 = exp2_hw(d1);
      s += w0;
      s1 += w1;
      if (ENT) {
        t = fmaf(w0, fmaxf(d0, kClampD), t);
        t1 = fmaf(w1, fmaxf(d1, kClampD), t1);
      }
    }
    s += s1;
    if (ENT) t += t1;
  }
};

// (m, r, u) of the union of R sets with those of their own, one a lane (r = -1: an empty set)
template <int R>
__device__ __forceinline__ void join_sets(float& m, float& r, float& u, float c) {
  const float top = gmax<R>(m), ref = top == -INFINITY ? 0.f : top;
  const float shift = fmaxf((m - ref) * c, kClampD), f = exp2_hw(shift);
  const bool holds = m == top && m != -INFINITY;
  const float others = rsum<R>(holds ? r : f * (1.f + r));
  u = rsum<R>(f * (u - (1.f + r) * shift));
  r = others + (rsum<R>(holds ? 1.f : 0.f) - 1.f);
  m = top;
}

// Joins the threads' partial results; on return (m, r, u) are the same in every thread.
//   resum(holder): sum over x < m of 2^(c (x - m)) over this thread's share of the elements that thread `holder` had
template <int NT>
struct JoinShared {
  f32x4 wave[NT / 64];
  float again[NT / 64];
};
template <int NT, bool ENT, typename ReSum>
__device__ __forceinline__ void block_join(const Online& on, float c, JoinShared<NT>& sh, float& m, float& r, float& u, ReSum resum) {
  constexpr int W = NT / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float wm = gmax<64>(on.m), wref = wm == -INFINITY ? 0.f : wm;
  const float shift = fmaxf((on.m - wref) * c, kClampD), f = exp2_hw(shift);
  const bool holds = on.m == wm;
  const unsigned long long who = __ballot(holds);
  const float a = rsum<64>(holds ? on.s - 1.f : on.s * f), b = ENT ? -rsum<64>(f * fmaf(on.s, shift, on.t)) : 0.f;
  if (lane == 0) sh.wave[wave] = f32x4{wm, wm == -INFINITY && a == a ? -1.f : a + ((float)__popcll(who) - 1.f), b,
                                       __int_as_float(wave * 64 + __ffsll(who) - 1)};
  __syncthreads();
  const f32x4 mine = sh.wave[lane & (W - 1)];
  m = mine[0], r = mine[1], u = mine[2];
  join_sets<W>(m, r, u, c);
  if (m == -INFINITY && r == r) r = -1.f;          // nothing of non-zero probability
  else if (r < kNearCertain) {                     // one thread holds the largest: its sum has rounded the rest away
    const int w = __ffsll(__ballot(mine[0] == m)) - 1, holder = __float_as_int(__shfl(mine[3], w));
    const float mshift = fmaxf((on.m - m) * c, kClampD);
    const float again = rsum<64>(resum(holder, m) + ((int)threadIdx.x == holder ? 0.f : on.s * exp2_hw(mshift)));
    if (lane == 0) sh.again[wave] = again;
    __syncthreads();
    r = rsum<W>(sh.again[lane & (W - 1)]);
  }
}

constexpr int kRowThreads = 256;
constexpr int kWideThreads = 1024;      // few rows
constexpr int64_t kSingleRows = 4096, kSingleSlots = 2048;     // many rows of moderate length: one wavefront each
constexpr int kUnroll = 4;              // slots in flight per thread
constexpr int kGroups = 8;              // slot groups whose maxima a thread keeps for the selection
constexpr int kCand = 512;              // candidates of a selection

constexpr int kCandPad = 128;

constexpr int kMaxima = 4;              // largest values a lane holds in the search for the bound: 256 in all
template <int NT>
struct TopShared {
  float gm[kGroups][NT];               // largest value of a thread's slot group
  float tmax[NT < 256 ? 256 : NT];
  uint16_t list[kGroups * NT];
  cand_t cand[kCand + kCandPad];
  int groups, count;
  uint32_t tau;
  cand_t best[NT / 64];
  int scan[NT / 64];
};

// largest t with count(key >= t) >= k over the wavefront's G keys a lane (0 if there are fewer), or a smaller one that not
// many more than k keys reach: bit by bit, down to the bits that differ between values of the type.  `top` is the largest
// key: most often k keys share its exponent, and the search starts below that.
template <int DT, int G>
__device__ __forceinline__ uint32_t lower_bound_of(const uint32_t* g, uint32_t top, int k) {
  auto count = [&](uint32_t t) {
    int c = 0;
#pragma unroll
    for (int w = 0; w < G; ++w) c += __popcll(__ballot(g[w] >= t));
    return c;
  };
  const uint32_t start = top & 0xff800000u;
  int c = count(start);
  uint32_t tau = c >= k ? start : 0u;
  const int enough = k + (k >> 2) + 1;
  for (int bit = c >= k ? 22 : 31; bit >= Elem<DT>::kOpenBits && !(tau != 0u && c <= enough); --bit) {
    const uint32_t t = tau | (1u << bit);
    const int ct = count(t);
    if (ct >= k) {
      tau = t;
      c = ct;
    }
  }
  return tau;
}

// Ranks the `have` candidates of a list with room for kCandPad more by counting the better ones, and emits those of rank
// below k.  Few candidates are counted by up to 16 lanes each: have^2 / NT comparisons a thread.
template <int NT, typename Emit>
__device__ __forceinline__ void rank_candidates(cand_t* cand, int have, int k, Emit emit) {
  const int tid = threadIdx.x;
  for (int i = tid; i < kCandPad; i += NT) cand[have + i] = 0;
  __syncthreads();
  int sh = 0;
  while (sh < 4 && (have << (sh + 1)) <= NT) ++sh;
  const int lanes = 1 << sh, sub = tid & (lanes - 1);
  for (int i0 = 0; i0 < have; i0 += NT >> sh) {
    const int i = i0 + (tid >> sh);
    const cand_t me = i < have ? cand[i] : 0;
    int rank = 0;
    for (int j = sub; j < have; j += 8 * lanes) {
      cand_t o[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) o[q] = cand[j + q * lanes];      // past the end: 0, better than nothing
#pragma unroll
      for (int q = 0; q < 8; ++q) rank += o[q] > me ? 1 : 0;
    }
    if (sh >= 1) rank += (int)dpp_move_u<0xB1>((uint32_t)rank);
    if (sh >= 2) rank += (int)dpp_move_u<0x4E>((uint32_t)rank);
    if (sh >= 3) rank += (int)dpp_move_u<0x141>((uint32_t)rank);
    if (sh >= 4) rank += (int)dpp_move_u<0x140>((uint32_t)rank);
    if (i < have && sub == 0 && rank < k) emit(rank, (uint32_t)(me >> 32), (int)~(uint32_t)me);
  }
}

// The selection's result goes through `emit(rank, key, index)`.
//
// Every thread knows the largest value of each of its slot groups.  tau, at most the k-th largest of the largest values of
// 256 threads (or sets of threads), is a lower bound of the k-th largest element, so only groups whose largest value
// reaches tau hold any of the k: these are listed, read again with a slot per thread, and the elements that reach tau -
// little more than k in an ordinary row - are ranked by counting.  Rows with more candidates than fit (many equal values)
// take the ordered scan below, and in the worst case one pass over the listed groups per rank.
template <int DT, int VEC, int NT, typename Emit>
__device__ void block_top(TopShared<NT>& sh, const char* p, const Span<VEC>& span, int s0, int s1, int gsz, int k, float m, float tmax,
                          Emit emit) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int groups = (s1 - s0 + NT * gsz - 1) / (NT * gsz);
  if (tid == 0) sh.count = sh.groups = 0;
  if constexpr (NT == 64) {      // a wavefront by itself: four sets of its slot groups
#pragma unroll
    for (int w = 0; w < kMaxima; ++w) {
      const float a = w < groups ? sh.gm[w][tid] : -INFINITY, b = w + kMaxima < groups ? sh.gm[w + kMaxima][tid] : -INFINITY;
      sh.tmax[64 * w + lane] = fmaxf(a, b);
    }
  } else {
    sh.tmax[tid] = tmax;
  }
  __syncthreads();
  if (tid < 64) {          // one wavefront searches: the others would only contend with it
    uint32_t g[kMaxima];
#pragma unroll
    for (int w = 0; w < kMaxima; ++w) {
      float t = sh.tmax[64 * w + lane];
#pragma unroll
      for (int j = kMaxima; j < NT / 64; j += kMaxima) t = fmaxf(t, sh.tmax[64 * (w + j) + lane]);
      g[w] = order_key(t);
    }
    const uint32_t t = lower_bound_of<DT, kMaxima>(g, order_key(m), k);
    if (lane == 0) sh.tau = t <= kKeyMinusInf ? kKeyMinusInf + 1 : t;      // -inf is no alternative
  }
  uint32_t gk[kGroups];
#pragma unroll
  for (int q = 0; q < kGroups; ++q) gk[q] = order_key(q < groups ? sh.gm[q][tid] : -INFINITY);
  __syncthreads();
  uint32_t tau = sh.tau;
  // the groups with a value that reaches `lowest`, in sh.list
  auto list_groups = [&](uint32_t lowest) {
    if (order_key(tmax) >= lowest) {
#pragma unroll
      for (int q = 0; q < kGroups; ++q)
        if (gk[q] >= lowest) sh.list[atomicAdd(&sh.groups, 1)] = (uint16_t)(q * NT + tid);
    }
    __syncthreads();
  };
  // f(keys that reach `lowest`, index of the slot's first element, bits of those elements) for the listed groups, until done()
  auto each_slot = [&](uint32_t lowest, auto done, auto f) {
    const int total = sh.groups * gsz;
    for (int j = tid; j < total && !done(); j += NT) {
      const int l = j / gsz, at = sh.list[l];
      const int s = s0 + (at & (NT - 1)) + NT * (at / NT * gsz + (j - l * gsz));
      if (s >= s1) continue;
      float v[VEC];
      const int b = span.base(s);
      slot_load<DT, VEC>(p, b, v);
      uint32_t key[VEC], bits = 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        key[e] = order_key(v[e]);
        if (span.holds(s, b + e) && key[e] >= lowest) bits |= 1u << e;
      }
      if (bits) f(key, b, bits);
    }
  };
  // (stops where there are more than fit: a row of equal values would add all of its slots to one counter, 300 us instead
  // of 59 for 2048 x 65536 bfloat16)
  auto collect = [&](uint32_t lowest) {
    list_groups(lowest);
    const volatile int* count = &sh.count;
    each_slot(lowest, [&] { return *count > kCand; }, [&](const uint32_t* key, int b, uint32_t bits) {
      int at = atomicAdd(&sh.count, __popc(bits));
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if ((bits >> e) & 1u) {
          if (at < kCand) sh.cand[at] = candidate(key[e], (uint32_t)(b + e));
          ++at;
        }
    });
    __syncthreads();
    return sh.count;
  };
  // of many candidates those that can be among the k best: ranking takes the square of their number.  (Rows that fill few
  // of the threads' slot groups have no close bound: 5000 x (1 .. 2049) bfloat16, 64 alternatives 36 us, 107 without.)
  auto thin_out = [&](int have) {
    constexpr int MINE = (kCand + NT - 1) / NT;
    cand_t mine[MINE];
    __syncthreads();          // every wavefront has read the number of candidates, which is counted again
#pragma unroll
    for (int q = 0; q < MINE; ++q) mine[q] = tid + NT * q < have ? sh.cand[tid + NT * q] : 0;
    if (tid < 64) {
      uint32_t g[kCand / 64];
#pragma unroll
      for (int w = 0; w < kCand / 64; ++w) g[w] = 64 * w + lane < have ? (uint32_t)(sh.cand[64 * w + lane] >> 32) : 0u;
      const uint32_t t = lower_bound_of<DT, kCand / 64>(g, order_key(m), k);
      if (lane == 0) sh.tau = t, sh.count = 0;
    }
    __syncthreads();
    const uint32_t least = sh.tau;
#pragma unroll
    for (int q = 0; q < MINE; ++q)
      if (tid + NT * q < have && (uint32_t)(mine[q] >> 32) >= least) sh.cand[atomicAdd(&sh.count, 1)] = mine[q];
    __syncthreads();
    return sh.count;
  };
  int have = collect(tau);
  int done;
  if (have <= kCand) {
    if (have > 2 * k + 64) have = thin_out(have);
    rank_candidates<NT>(sh.cand, have, k, emit);
    done = have;
  } else {
    // many values reach tau: make it the key of the k-th largest of the threads' values itself (where k threads have
    // one), so that those equal to it can be told from those above
    uint32_t g[kMaxima];
#pragma unroll
    for (int w = 0; w < kMaxima; ++w) {
      float t = sh.tmax[64 * w + lane];
#pragma unroll
      for (int j = kMaxima; j < NT / 64; j += kMaxima) t = fmaxf(t, sh.tmax[64 * (w + j) + lane]);
      g[w] = order_key(t);
    }
    auto reach = [&](uint32_t t) {
      int c = 0;
#pragma unroll
      for (int w = 0; w < kMaxima; ++w) c += __popcll(__ballot(g[w] >= t));
      return c;
    };
    for (uint32_t t = tau; reach(t) >= k;) {       // the next of the threads' values, as long as k reach it
      uint32_t next = 0xffffffffu;
#pragma unroll
      for (int w = 0; w < kMaxima; ++w) next = (g[w] >= t && g[w] < next) ? g[w] : next;
      next = ~gmax_u<64>(~next);
      if (reach(next) < k) break;
      tau = next;
      t = next + 1u;
    }
    const uint32_t above = tau + 1u;
    __syncthreads();
    if (tid == 0) sh.count = sh.groups = 0;
    __syncthreads();
    have = collect(above);
    if (have <= kCand) {
      rank_candidates<NT>(sh.cand, have, k, emit);
      done = have < k ? have : k;
      // elements equal to tau, lowest index first: a round covers NT consecutive slots, in index order by thread
      for (int it = 0; done < k && s0 + NT * it < s1; ++it) {
        const int s = s0 + tid + NT * it;
        uint32_t bits = 0;
        const int b = span.base(s < s1 ? s : s1 - 1);
        if (s < s1) {
          float v[VEC];
          slot_load<DT, VEC>(p, b, v);
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (span.holds(s, b + e) && order_key(v[e]) == tau) bits |= 1u << e;
        }
        int run = __popc(bits);     // inclusive scan over the wavefront
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const int up = __shfl_up(run, off);
          if (lane >= off) run += up;
        }
        __syncthreads();
        if (lane == 63) sh.scan[tid >> 6] = run;
        __syncthreads();
        int before = run - __popc(bits), total = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) {
          if (w < (tid >> 6)) before += sh.scan[w];
          total += sh.scan[w];
        }
        int rank = done + before;
        for (int e = 0; e < VEC; ++e)
          if ((bits >> e) & 1u) {
            if (rank < k) emit(rank, tau, b + e);
            ++rank;
          }
        done += total;
      }
    } else {
      // one rank per pass: the best (key, lower index) after the last one
      cand_t last = ~0ull;
      for (done = 0; done < k; ++done) {
        cand_t best = 0;
        each_slot(above, [] { return false; }, [&](const uint32_t* key, int b, uint32_t bits) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const cand_t o = candidate(key[e], (uint32_t)(b + e));
            if (((bits >> e) & 1u) && o < last && o > best) best = o;
          }
        });
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
          const cand_t o = __shfl_xor(best, off);
          best = o > best ? o : best;
        }
        __syncthreads();
        if (lane == 0) sh.best[tid >> 6] = best;
        __syncthreads();
        for (int w = 0; w < NT / 64; ++w) best = sh.best[w] > best ? sh.best[w] : best;
        if (best == 0) break;
        last = best;
        if (tid == 0) emit(done, (uint32_t)(best >> 32), (int)~(uint32_t)best);
      }
    }
  }
  for (int j = done + tid; j < k; j += NT) emit(j, 0u, -1);
}

// One workgroup per row (or per part of a row): every element is read once, kUnroll 16-byte slots in flight per thread.
// Four wavefronts where there are rows or parts enough to fill the chip (several workgroups a compute unit hide each
// other's joins), sixteen where there are few, one where there are many of moderate length.  Measured: 2048 x 65536
// bfloat16, log-probability alone 54 us (5.0 TB/s), with entropy and 8 alternatives 66 us (4.1 TB/s; the vector units are
// 81 % busy); float32 92 us (5.8 TB/s) and 101 us; 8192 x 4096 bfloat16 15 and 26 us; 50 x 50000 float32 with 64
// alternatives 15 us, bound by the latency of its phases.  Loading a round ahead gained nothing.
template <int DT, bool ENT, bool TOP, int NT>
__global__ void __launch_bounds__(NT) k_cat_fwd_row(Fwd a) {
  constexpr int VEC = Elem<DT>::N, ES = sizeof(typename Elem<DT>::type);
  __shared__ JoinShared<NT> join;
  __shared__ typename std::conditional<TOP, TopShared<NT>, int>::type top_sh;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x - (int)(row * a.parts);
  const bool seen = row_seen(a.r, row);
  if (!seen && !ENT && !TOP) {
    if (tid == 0 && part == 0 && a.log_prob) a.log_prob[row] = 0.f;
    return;
  }
  if (!ENT && !TOP && a.weight && a.weight[wrap(row, a.w_period, a.r.rows)] == 0.f) return;
  const int n = row_size(a.r, row);
  const char* p = a.r.x + row * a.r.ld * ES;
  const Span<VEC> span(p, ES, a.r.V, n);
  const int ns = span.slots, per = ((ns + a.parts - 1) / a.parts + 15) & ~15;      // equal to 16 slots
  const int s0 = part * per < ns ? part * per : ns, s1 = s0 + per < ns ? s0 + per : ns;
  int gsz = (s1 - s0 + NT * kGroups - 1) / (NT * kGroups);    // slots per group of the selection: 1, 2 or whole rounds
  gsz = gsz <= 2 ? (gsz < 1 ? 1 : gsz) : (gsz + kUnroll - 1) / kUnroll * kUnroll;
  Online on;
  float gmx = -INFINITY;
  int in_group = 0, group = 0;
  const int groups = (s1 - s0 + NT * gsz - 1) / (NT * gsz);
  // IN slots in flight per thread, kUnroll at a time through the sums
  constexpr int IN = NT == kWideThreads ? 2 * kUnroll : kUnroll;
  for (int sb = s0 + tid; sb < s1; sb += NT * IN) {
    Raw16 raw[IN];
#pragma unroll
    for (int q = 0; q < IN; ++q) {
      const int sq = sb + q * NT;
      raw[q] = *(const Raw16*)(p + (int64_t)span.base(sq < s1 ? sq : sb) * ES);
    }
#pragma unroll
    for (int h = 0; h < IN; h += kUnroll) {
      const int s = sb + h * NT;
      // the wavefront's first slot: a last round sums only as many slots a lane as it has
      const int first = __builtin_amdgcn_readfirstlane(s);
      const bool full = first + (kUnroll - 1) * NT < s1;
      float v[kUnroll * VEC];
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        Elem<DT>::unpack(raw[h + q], v + q * VEC);
        const int sq = s + q * NT;
        if (sq >= s1 || !span.whole(sq)) {       // the row's first and last slots, and past the end
          const int b = span.base(sq);
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (sq >= s1 || !span.holds(sq, b + e)) v[q * VEC + e] = -INFINITY;
        }
      }
      float mx;
      if constexpr (TOP) {
        float part[kUnroll];
#pragma unroll
        for (int q = 0; q < kUnroll; ++q) part[q] = max_of<VEC>(v + q * VEC, -INFINITY);
        const float half0 = max3(part[0], part[1], part[1]), half1 = max3(part[2], part[3], part[3]);
        mx = max3(half0, half1, half1);
        static_assert(kUnroll == 4, "");
        if (gsz >= kUnroll) {
          if (s < s1) {
            gmx = max3(mx, gmx, gmx);
            in_group += kUnroll;
            if (in_group == gsz) {
              top_sh.gm[group++][tid] = gmx;
              gmx = -INFINITY;
              in_group = 0;
            }
          }
        } else {
          const int left = groups - group;       // (groups past the last one have no slots)
          if (gsz == 1) {
#pragma unroll
            for (int q = 0; q < kUnroll; ++q)
              if (q < left) top_sh.gm[group + q][tid] = part[q];
            group += kUnroll;
          } else {
            if (0 < left) top_sh.gm[group][tid] = half0;
            if (1 < left) top_sh.gm[group + 1][tid] = half1;
            group += 2;
          }
        }
      } else {
        mx = max_of<kUnroll * VEC>(v, -INFINITY);
      }
      if (full) {
        on.template add<kUnroll * VEC, ENT>(v, mx, a.c);
      } else {
#pragma unroll
        for (int q = 0; q < kUnroll; ++q)
          if (first + q * NT < s1) on.template add<VEC, ENT>(v + q * VEC, max_of<VEC>(v + q * VEC, -INFINITY), a.c);
      }
    }
  }
  if constexpr (TOP) {
    for (; group < groups; ++group) {
      top_sh.gm[group][tid] = gmx;
      gmx = -INFINITY;
    }
  }
  float m, r, u;
  block_join<NT, ENT>(on, a.c, join, m, r, u, [&](int h, float ref) {
    float sum = 0.f;
    for (int s = s0 + h + NT * tid; s < s1; s += NT * NT) {
      float v[VEC];
      const int b = span.base(s);
      slot_load<DT, VEC>(p, b, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (span.holds(s, b + e) && v[e] < ref) sum += exp2_hw((v[e] - ref) * a.c);
    }
    return sum;
  });
  const bool empty = m == -INFINITY && r == -1.f;
  if (a.part) {
    if (tid == 0) a.part[row * a.parts + part] = f32x4{m, r, u, 0.f};
    if constexpr (TOP) {
      uint2* o = a.part_top + (row * a.parts + part) * a.top;
      block_top<DT, VEC, NT>(top_sh, p, span, s0, s1, gsz, a.top, m, on.m,
                         [&](int rank, uint32_t key, int i) { o[rank] = make_uint2(key, (uint32_t)i); });
    }
    return;
  }
  const float logs = empty ? 0.f : log1p_row(r), inv_s = empty ? 0.f : __builtin_amdgcn_rcpf(1.f + r);
  const float H = empty ? 0.f : logs + kLn2 * u * inv_s;
  if (tid == 0) {
    if (a.log_prob) {
      float lp = 0.f;
      if (seen) {
        const int64_t X = a.r.X[wrap(row, a.r.x_period, a.r.rows)];
        lp = empty ? -INFINITY : ((X < 0 || X >= n) ? NAN : (Elem<DT>::load(p, X) - m) - logs);
      }
      a.log_prob[row] = lp;
    }
    if (a.entropy) a.entropy[row] = H;
    if (a.stats) a.stats[row] = f32x4{m, inv_s, logs, H};
  }
  if constexpr (TOP) {
    if (logs != logs) {
      for (int j = tid; j < a.top; j += NT) {
        a.top_idx[row * a.top + j] = -1;
        a.top_lp[row * a.top + j] = NAN;
      }
      return;
    }
    block_top<DT, VEC, NT>(top_sh, p, span, s0, s1, gsz, a.top, m, on.m, [&](int rank, uint32_t key, int i) {
      a.top_idx[row * a.top + rank] = i;
      a.top_lp[row * a.top + rank] = i < 0 ? -INFINITY : (key_value(key) - m) - logs;
    });
  }
}

// (m, r, u) of a row from its parts (every wavefront, a lane per part)
__device__ __forceinline__ void join_parts(const f32x4* part, int parts, float c, float& m, float& r, float& u) {
  const int lane = threadIdx.x & 63;
  const f32x4 me = lane < parts ? part[lane] : f32x4{-INFINITY, -1.f, 0.f, 0.f};
  m = me[0], r = me[1], u = me[2];
  join_sets<64>(m, r, u, c);
}

// The parts' ordered lists hold parts * k candidates.  Where the j-th keys of ceil(k / j) parts reach tau, k elements do: tau
// is the largest such bound over j = 1, 2, 4 .. k, whatever few parts hold the large values (a row's last part may have a
// few elements, and with sizes most parts none).  Those that reach it are ranked by counting.  (8 x 262147 float32, 64
// alternatives: 26 us a call; by the smallest of the parts' ceil(k / parts)-th keys 1100, nearly all 4096 to rank.)
constexpr int kJoinThreads = 256;
constexpr int kJoinDepths = 7;      // j = 1 .. 64
static_assert(kMaxTop <= 1 << (kJoinDepths - 1), "");
template <int DT>
__global__ void __launch_bounds__(kJoinThreads) k_cat_fwd_join(Fwd a) {
  __shared__ cand_t cand[kMaxParts * kMaxTop + kCandPad];
  __shared__ int count, sums[2][kJoinThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const bool seen = row_seen(a.r, row);
  if (!seen && !a.entropy && !a.top) return;        // the parts' launch has written it
  const int n = row_size(a.r, row);
  const char* p = a.r.x + row * a.r.ld * (int64_t)sizeof(typename Elem<DT>::type);
  float m, r, u;
  join_parts(a.part + row * a.parts, a.parts, a.c, m, r, u);
  const bool empty = m == -INFINITY && !(r != r);
  const float logs = empty ? 0.f : log1p_row(r), inv_s = empty ? 0.f : __builtin_amdgcn_rcpf(1.f + r);
  const float H = empty ? 0.f : logs + kLn2 * u * inv_s;
  if (tid == 0) {
    count = 0;
    if (a.log_prob) {
      float lp = 0.f;
      if (seen) {
        const int64_t X = a.r.X[wrap(row, a.r.x_period, a.r.rows)];
        lp = empty ? -INFINITY : ((X < 0 || X >= n) ? NAN : (Elem<DT>::load(p, X) - m) - logs);
      }
      a.log_prob[row] = lp;
    }
    if (a.entropy) a.entropy[row] = H;
    if (a.stats) a.stats[row] = f32x4{m, inv_s, logs, H};
  }
  if (!a.top) return;
  if (logs != logs) {
    for (int j = tid; j < a.top; j += kJoinThreads) {
      a.top_idx[row * a.top + j] = -1;
      a.top_lp[row * a.top + j] = NAN;
    }
    return;
  }
  const uint2* list = a.part_top + row * a.parts * a.top;
  uint32_t jth[kJoinDepths], tau = 1u;  // (key 0: past the end of a part's list)
#pragma unroll
  for (int q = 0; q < kJoinDepths; ++q) {
    const int j = 1 << q < a.top ? 1 << q : a.top;
    jth[q] = lane < a.parts ? list[lane * a.top + j - 1].x : 0u;
  }
#pragma unroll
  for (int q = 0; q < kJoinDepths; ++q) {
    const int j = 1 << q < a.top ? 1 << q : a.top, need = (a.top + j - 1) / j;
    if (need > a.parts || (q > 0 && 1 << (q - 1) >= a.top)) continue;
    tau = max(tau, lower_bound_of<DT, 1>(jth + q, gmax_u<64>(jth[q]), need));
  }
  __syncthreads();
  for (int j = tid; j < a.parts * a.top; j += kJoinThreads) {
    const uint2 o = list[j];
    if (o.x >= tau) cand[atomicAdd(&count, 1)] = candidate(o.x, o.y);
  }
  __syncthreads();
  int have = count;
  if (have > 4 * a.top + 64) {
    // many equal values: what reaches the k-th largest candidate or a smaller one, key and index bit by bit (8 x 262147
    // float32 zeros, 64 alternatives: 52 us a call, 1150 with all of them ranked)
    constexpr int MINE = kMaxParts * kMaxTop / kJoinThreads;
    cand_t mine[MINE], least = 0;
#pragma unroll
    for (int q = 0; q < MINE; ++q) mine[q] = tid + kJoinThreads * q < have ? cand[tid + kJoinThreads * q] : 0;
    for (int bit = 63, reach = have; bit >= 0 && reach > 2 * a.top; --bit) {
      const cand_t t = least | 1ull << bit;
      uint32_t n = 0;
#pragma unroll
      for (int q = 0; q < MINE; ++q) n += mine[q] >= t ? 1u : 0u;
      n = rsum_u<64>(n);
      if (lane == 0) sums[bit & 1][tid >> 6] = (int)n;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int w = 0; w < kJoinThreads / 64; ++w) all += sums[bit & 1][w];
      if (all >= a.top) least = t, reach = all;
    }
    __syncthreads();
    if (tid == 0) count = 0;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < MINE; ++q)
      if (mine[q] && mine[q] >= least) cand[atomicAdd(&count, 1)] = mine[q];
    __syncthreads();
    have = count;
  }
  rank_candidates<kJoinThreads>(cand, have, a.top, [&](int rank, uint32_t key, int i) {
    a.top_idx[row * a.top + rank] = i;
    a.top_lp[row * a.top + rank] = (key_value(key) - m) - logs;
  });
  for (int j = have + tid; j < a.top; j += kJoinThreads) {
    a.top_idx[row * a.top + j] = -1;
    a.top_lp[row * a.top + j] = -INFINITY;
  }
}

// A slot of a chunk: the last slot of a row overlaps the one before it, which may be another workgroup's, so only its own
// elements are written.
template <int DT>
__device__ __forceinline__ void chunk_store(char* out, int s, int base, const float* o) {
  constexpr int VEC = Elem<DT>::N;
  if (base == s * VEC) {
    slot_store<DT, VEC>(out, base, o);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (base + e >= s * VEC) Elem<DT>::store(out, base + e, o[e]);
  }
}

// Gradient of long rows: a workgroup per chunk of a row (kChunkSlots slots), the row's statistics are known.  One read and one
// write of the row: 1024 x 50001 float16 36 us (5.7 TB/s), 2048 x 65536 bfloat16 99 us (5.4 TB/s), as fast as a copy.
constexpr int kChunkSlots = kRowThreads * kUnroll;
template <int DT>
__global__ void __launch_bounds__(kRowThreads) k_cat_bwd_chunk(Bwd a) {
  constexpr int NT = kRowThreads, VEC = Elem<DT>::N, ES = sizeof(typename Elem<DT>::type);
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / a.chunks;
  const int s0 = (blockIdx.x - (int)(row * a.chunks)) * kChunkSlots;
  const int n = row_size(a.r, row), V = a.r.V;
  const int ns = (V + VEC - 1) / VEC;
  int64_t X;
  float gl;
  const RowGrad g = row_grad<64>(a, row, tid & 63, n, X, gl);
  const bool live = (g.S != 0.f || g.gh != 0.f || a.g_top) && g.inv_s != 0.f;
  const char* p = a.r.x + row * a.r.ld * ES;
  char* out = (char*)a.d + row * a.ld_d * ES;
  float v[kUnroll][VEC];
  if (live) {
#pragma unroll
    for (int q = 0; q < kUnroll; ++q) {
      const int s = s0 + tid + q * NT;
      slot_load<DT, VEC>(p, slot_base<VEC>(s < ns ? s : ns - 1, V), v[q]);
    }
  }
#pragma unroll
  for (int q = 0; q < kUnroll; ++q) {
    const int s = s0 + tid + q * NT;
    if (s >= ns) break;
    const int b = slot_base<VEC>(s, V);
    float o[VEC];
    if (live) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = g.dense(v[q][e]);
      if (b + VEC > n) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (b + e >= n) o[e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = 0.f;
    }
    chunk_store<DT>(out, s, b, o);
  }
  if (!live) return;
  __syncthreads();          // the dense part before the few categories written again
  const int64_t lo = (int64_t)s0 * VEC, hi = lo + (int64_t)kChunkSlots * VEC;
  const int entries = 1 + (a.g_top ? a.top : 0);
  for (int j = tid; j < entries; j += NT) {
    const int64_t v0 = j == 0 ? X : a.top_idx[row * a.top + j - 1];
    if (v0 < lo || v0 >= hi || v0 >= n) continue;
    Elem<DT>::store(out, v0, g.at(Elem<DT>::load(p, v0), own_share(a, row, v0, X, gl)));
  }
}


// The teacher's distribution over one row by a workgroup, entry j on thread j (the launch has k <= NT): p and log p of this
// thread's entry (p = 0 where it does not count), its index (-1), and what holds for the row.
struct TeacherEntry {
  float p, lp;
  int i;
  bool any, bad;
};
template <int NT>
__device__ __forceinline__ TeacherEntry teacher_row(const Teacher& t, int64_t row, int64_t rows, int n, BlockRed<NT>& red) {
  TeacherEntry e{0.f, 0.f, -1, false, false};
  float x = -INFINITY;
  bool bad = false;
  if ((int)threadIdx.x < t.k) {
    const int64_t at = wrap(row, t.t_period, rows) * t.k + threadIdx.x;
    const int64_t i = t.idx[at];
    const float v = teacher_logit(t, at);
    if (entry_counts(v, i)) {
      bad = i >= n || !(v < INFINITY);
      x = bad ? -INFINITY : v;
      e.i = bad ? -1 : (int)i;
    }
  }
  const float tm = block_max<NT>(x, red);
  const bool counts = e.i >= 0;
  float s = counts && x < tm ? exp2_hw((x - tm) * t.c) : 0.f, held = counts && x == tm ? 1.f : 0.f, b = bad ? 1.f : 0.f;
  block_sum3<NT>(s, held, b, red);
  e.bad = b > 0.f;
  e.any = held > 0.f || e.bad;
  if (counts) {
    e.lp = (x - tm) * t.inv_T - log1p_row(s + (held - 1.f));
    e.p = exp_hw(e.lp);
  }
  return e;
}

struct SparseShared {
  float p[kMaxTeacher];
  int i[kMaxTeacher];
};
// log of all of the teacher's probability on entry e's category, which may be given more than once: the same for each of
// its entries
__device__ __forceinline__ float share_of(const SparseShared& sh, int k, const TeacherEntry& e) {
  float p = 0.f;
  int same = 0;
  for (int j = 0; j < k; ++j)
    if (sh.i[j] == e.i) p += sh.p[j], ++same;
  return same > 1 ? logf(p) : e.lp;
}

// Loss and gradient of a row that fits the registers of one workgroup (NV slots per thread): the row is read once.  2048 x
// 65536 bfloat16 with 32 entries 118 us (4.5 TB/s read and written; two workgroups of 512 a compute unit, one of 1024 took
// 136), 4096 x 32000 106 us (5.0 TB/s), 1024 x 65536 float32 122 us (4.4 TB/s: one workgroup of 1024 a compute unit, whose
// loads, sums and stores do not overlap).
template <int DT, int NT, int NV>
__global__ void __launch_bounds__(NT) k_cat_distill_row(Dist a) {
  constexpr int VEC = Elem<DT>::N, ES = sizeof(typename Elem<DT>::type);
  __shared__ BlockRed<NT> red;
  __shared__ JoinShared<NT> join;
  __shared__ SparseShared sp;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int V = a.r.V, ns = (V + VEC - 1) / VEC;
  char* out = (char*)a.d + row * a.ld_d * ES;
  const float w = a.t.weight ? a.t.weight[wrap(row, a.t.w_period, a.r.rows)] : 1.f;
  auto zeros = [&]() {
    const float z[VEC] = {};
    for (int s = tid; s < ns; s += NT) slot_store<DT, VEC>(out, slot_base<VEC>(s, V), z);
  };
  if (w == 0.f) {
    if (tid == 0) {
      if (a.per_row) a.per_row[row] = 0.f;
      a.loss_part[row] = 0.0;
    }
    if (a.d) zeros();
    return;
  }
  const char* p = a.r.x + row * a.r.ld * ES;
  const int n = row_size(a.r, row);
  const Span<VEC> span(p, ES, V, V);
  const int slots = span.slots;
  // a wavefront takes part in as many of the NV rounds as it has slots
  const int wave0 = __builtin_amdgcn_readfirstlane(tid);
  auto has = [&](int q) { return wave0 + NT * q < slots; };
  u32x4 raw[NV];
#pragma unroll
  for (int q = 0; q < NV; ++q)
    if (has(q)) {
      const int s = tid + NT * q;
      raw[q] = __builtin_bit_cast(u32x4, *(const Raw16*)(p + (uint32_t)(span.base(s < slots ? s : slots - 1) * ES)));
    }
  const TeacherEntry te = teacher_row<NT>(a.t, row, a.r.rows, n, red);
  const float xi = te.i >= 0 ? Elem<DT>::load(p, te.i) : 0.f;
  // what does not count becomes -inf, once: past the row's size, and what a first or last slot shares with its neighbour
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    if (!has(q)) break;
    if ((q > 0 || span.lead == 0) && NT * (q + 1) * VEC - span.lead <= n) continue;      // a round of whole slots
    const int s = again(tid) + NT * q;
    if (s >= slots || !span.whole(s) || span.base(s) + VEC > n) {
      const int b = span.base(s < slots ? s : slots - 1);
      float v[VEC];
      pass_over<DT>(raw[q], v);
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (!span.holds(s, b + e) || b + e >= n) v[e] = -INFINITY;
      Raw16 w;
      Elem<DT>::pack(v, w);
      raw[q] = __builtin_bit_cast(u32x4, w);
    }
  }
  Online on;
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    if (!has(q)) break;
    float v[VEC];
    pass_over<DT>(raw[q], v);
    on.m = max_of<VEC>(v, on.m);
  }
  const float local = on.m == -INFINITY ? 0.f : on.m;
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    if (!has(q)) break;
    float v[VEC];
    pass_over<DT>(raw[q], v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) on.s += exp2_hw((v[e] - local) * a.t.c);
  }
  asm volatile("" : "+v"(on.s));        // summed here, not where it is used
  float m, r, u;
  block_join<NT, false>(on, a.t.c, join, m, r, u, [&](int h, float ref) {
    float sum = 0.f;
    if (h == tid) {
#pragma unroll
      for (int q = 0; q < NV; ++q) {
        if (!has(q)) break;
        float v[VEC];
        pass_over<DT>(raw[q], v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum += v[e] < ref ? exp2_hw((v[e] - ref) * a.t.c) : 0.f;
      }
    }
    return sum;
  });
  const bool empty = m == -INFINITY && r == -1.f;
  const float logs = empty ? 0.f : log1p_row(r), inv_s = empty ? 0.f : __builtin_amdgcn_rcpf(1.f + r);
  const float lq = (xi - m) * a.t.inv_T - logs;
  float kl = (te.i >= 0 && te.p > 0.f && !empty) ? te.p * (te.lp - lq) : 0.f, z0 = 0.f, z1 = 0.f;
  if (tid < a.t.k) {
    sp.p[tid] = te.p;
    sp.i[tid] = te.i;
  }
  block_sum3<NT>(kl, z0, z1, red);
  if (te.any && empty) kl = INFINITY;
  if (te.bad) kl = NAN;
  if (tid == 0) {
    if (a.per_row) a.per_row[row] = kl;
    if (a.stats) a.stats[row] = f32x4{m, inv_s, logs, 0.f};
    a.loss_part[row] = (double)w * (double)kl;
  }
  if (!a.d) return;
  if (!te.any || (empty && !te.bad)) {
    zeros();
    return;
  }
  const float scale = te.bad ? NAN : w * a.t.inv_T, f = scale * inv_s;
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int s = again(tid) + NT * q;
    if (s >= slots) break;
    float v[VEC];
    pass_over<DT>(raw[q], v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = exp2_hw((v[e] - m) * a.t.c) * f;
    const int b = span.base(s);
    if (span.whole(s)) slot_store<DT, VEC>(out, b, v);
    else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (span.holds(s, b + e)) Elem<DT>::store(out, b + e, v[e]);
    }
  }
  __syncthreads();          // the dense part before what is written again
  if (!(fabsf(f) < INFINITY))        // past the row's size 0 all the same
    for (int i = n + tid; i < V; i += NT) Elem<DT>::store(out, i, 0.f);
  if (te.i >= 0 && !te.bad) Elem<DT>::store(out, te.i, scale * q_minus_p(lq, share_of(sp, a.t.k, te)));
}

// Rows that are read by several workgroups: their parts' statistics (k_cat_fwd_row) joined, and the loss.
template <int DT>
__global__ void __launch_bounds__(kRowThreads) k_cat_distill_join(Dist a) {
  constexpr int NT = kRowThreads, ES = sizeof(typename Elem<DT>::type);
  __shared__ BlockRed<NT> red;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const float w = a.t.weight ? a.t.weight[wrap(row, a.t.w_period, a.r.rows)] : 1.f;
  if (w == 0.f) {
    if (tid == 0) {
      if (a.per_row) a.per_row[row] = 0.f;
      a.loss_part[row] = 0.0;
    }
    return;
  }
  const int n = row_size(a.r, row);
  const char* p = a.r.x + row * a.r.ld * ES;
  const TeacherEntry te = teacher_row<NT>(a.t, row, a.r.rows, n, red);
  const float xi = te.i >= 0 ? Elem<DT>::load(p, te.i) : 0.f;
  float m, r, u;
  join_parts(a.part + row * a.parts, a.parts, a.t.c, m, r, u);     // every wavefront does the same
  const bool empty = m == -INFINITY && !(r != r);
  const float logs = empty ? 0.f : log1p_row(r), inv_s = empty ? 0.f : __builtin_amdgcn_rcpf(1.f + r);
  float kl = (te.i >= 0 && te.p > 0.f && !empty) ? te.p * (te.lp - ((xi - m) * a.t.inv_T - logs)) : 0.f, z0 = 0.f, z1 = 0.f;
  block_sum3<NT>(kl, z0, z1, red);
  if (te.any && empty) kl = INFINITY;
  if (te.bad) kl = NAN;
  if (tid == 0) {
    if (a.per_row) a.per_row[row] = kl;
    a.stats[row] = f32x4{m, inv_s, logs, 0.f};
    a.loss_part[row] = (double)w * (double)kl;
  }
}

// The gradient of rows whose statistics are known, a workgroup per chunk of a row at a time.
template <int DT>
__global__ void __launch_bounds__(kRowThreads) k_cat_distill_chunk(Dist a) {
  constexpr int NT = kRowThreads, VEC = Elem<DT>::N, ES = sizeof(typename Elem<DT>::type);
  __shared__ BlockRed<NT> red;
  __shared__ SparseShared sp;
  const float gs = a.gscale ? *a.gscale : 1.f;
  if (a.unless_one && gs == 1.f) return;
  const int tid = threadIdx.x;
  const int V = a.r.V, ns = (V + VEC - 1) / VEC;
  const int64_t items = a.r.rows * a.chunks;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t row = item / a.chunks;
    const int s0 = (int)(item - row * a.chunks) * kChunkSlots;
    const int n = row_size(a.r, row);
    const char* p = a.r.x + row * a.r.ld * ES;
    char* out = (char*)a.d + row * a.ld_d * ES;
    const float w = a.t.weight ? a.t.weight[wrap(row, a.t.w_period, a.r.rows)] : 1.f;
    bool live = w != 0.f;
    float v[kUnroll][VEC];
    TeacherEntry te{0.f, 0.f, -1, false, false};
    f32x4 st = {0.f, 0.f, 0.f, 0.f};
    if (live) {
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const int s = s0 + tid + q * NT;
        slot_load<DT, VEC>(p, slot_base<VEC>(s < ns ? s : ns - 1, V), v[q]);
      }
      st = a.stats[row];
      te = teacher_row<NT>(a.t, row, a.r.rows, n, red);
      if (tid < a.t.k) {
        sp.p[tid] = te.p;
        sp.i[tid] = te.i;
      }
      live = te.any && (st[1] != 0.f || te.bad);
    }
    const float scale = te.bad ? NAN : gs * w * a.t.inv_T, f = scale * st[1];
#pragma unroll
    for (int q = 0; q < kUnroll; ++q) {
      const int s = s0 + tid + q * NT;
      if (s < ns) {
        const int b = slot_base<VEC>(s, V);
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = live && b + e < n ? exp2_hw((v[q][e] - st[0]) * a.t.c) * f : 0.f;
        chunk_store<DT>(out, s, b, o);
      }
    }
    __syncthreads();        // the dense part, and sp, before the teacher's categories are written again
    const int64_t lo = (int64_t)s0 * VEC;
    if (live && !te.bad && te.i >= lo && te.i < lo + (int64_t)kChunkSlots * VEC) {
      const float lq = (Elem<DT>::load(p, te.i) - st[0]) * a.t.inv_T - st[2];
      Elem<DT>::store(out, te.i, scale * q_minus_p(lq, share_of(sp, a.t.k, te)));
    }
    __syncthreads();        // sp is free again
  }
}

// The loss: the workgroups' (or rows') shares summed in a fixed order.
constexpr int kLossThreads = 1024;
__global__ void __launch_bounds__(kLossThreads) k_cat_loss(const double* part, int64_t n, float* loss) {
  __shared__ double w[kLossThreads / 64];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += kLossThreads) s += part[i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < kLossThreads / 64; ++i) t += w[i];
    *loss = (float)t;
  }
}

// ------------------------------------------------------------------------------------------ host side

int check_rows(const DmvCatRows* r) {
  if (!r || r->rows < 0 || r->V < 1 || r->ld < 0) return DMV_E_BADARG;
  if (r->dtype < DMV_F32 || r->dtype > DMV_F16) return DMV_E_UNSUPPORTED;
  if (r->rows == 0) return DMV_OK;
  if (!r->logits || ((uintptr_t)r->logits % elem_size(r->dtype)) != 0) return DMV_E_BADARG;
  if ((r->X && r->x_period < 1) || (r->M && r->m_period < 1) || (r->sizes && r->size_period < 1)) return DMV_E_BADARG;
  // row numbers of short rows and threads of a launch (64 a row, whole workgroups) in 32 bits, slot numbers in 32 bits with
  // room for a chunk
  if (r->rows >= ((int64_t)1 << 26) - 4 || r->V > 0x7fffffff - (1 << 20)) return DMV_E_UNSUPPORTED;
  return DMV_OK;
}
bool fits_grid(int64_t groups, int threads) { return groups * threads < (int64_t)1 << 32; }
Rows rows_of(const DmvCatRows* r) {
  return Rows{(const char*)r->logits, r->ld, r->rows, r->V, r->X, r->M, r->sizes, r->x_period, r->m_period, r->size_period};
}

// Short rows: `f` gets the tag of the smallest register tile that holds V elements (up to 32 elements a lane; rows shorter
// than a 16-byte slot are read one element at a time).
template <int DT_, int VEC_, int L_, int SL_>
struct Tile {
  static constexpr int DT = DT_, VEC = VEC_, L = L_, SL = SL_;
  static int64_t groups(int64_t rows) { return (rows + kSmallThreads / L - 1) / (kSmallThreads / L); }
};
template <int DT, typename F>
void wide_tile(int V, int lanes, F f) {
  constexpr int N = Elem<DT>::N, S = 32 / N;
  const int ns = (V + N - 1) / N;
  if (lanes <= 8 && ns <= 8 * S) return f(Tile<DT, N, 8, S>());
  if (ns <= 16 * S) return f(Tile<DT, N, 16, S>());
  if (ns <= 32 * S) return f(Tile<DT, N, 32, S>());
  return f(Tile<DT, N, 64, S>());
}
template <int DT, typename F>
void small_tile(int V, F f) {
  constexpr int N = Elem<DT>::N, S = 32 / N;
  const int ns = (V + N - 1) / N;
  if (V < N) return f(Tile<DT, 1, 4, 2>());
  if (ns <= 4) return f(Tile<DT, N, 4, 1>());
  if (ns <= 8) return f(Tile<DT, N, 4, 2>());
  if (ns <= 16) return f(Tile<DT, N, 4, 4>());
  if constexpr (S == 8)
    if (ns <= 32) return f(Tile<DT, N, 4, 8>());
  wide_tile<DT>(V, 8, f);
}
// ... for distillation: a lane group's k teacher entries are in LDS, which 256 / L groups share
template <int DT, typename F>
void teacher_tile(int V, int k, F f) {
  if (k <= 64) return small_tile<DT>(V, f);
  if (V < Elem<DT>::N) return f(Tile<DT, 1, 16, 1>());
  wide_tile<DT>(V, k <= 128 ? 8 : 16, f);
}
// LDS of a workgroup's teacher entries
template <typename T>
size_t small_lds(int k) {
  return (size_t)(kSmallThreads / T::L) * k * sizeof(Entry);
}
template <typename F>
void by_type(int dt, F f) {
  if (dt == DMV_F32) f(std::integral_constant<int, DMV_F32>());
  else if (dt == DMV_BF16) f(std::integral_constant<int, DMV_BF16>());
  else f(std::integral_constant<int, DMV_F16>());
}

// Few rows: sixteen wavefronts to each, where four would have more than one round of loads.  (Eight for 300 to 1500 rows
// gained nothing: 1024 x 50000 float16 with entropy and 8 alternatives took 38 us instead of 29.)
bool wide_rows(int64_t groups, int V, int dt) { return groups <= 256 && V > kRowThreads * kUnroll * vec_elems(dt); }

// Many rows that are not very long: a wavefront to each.
bool single_wave_rows(int64_t groups, int V, int dt) { return groups >= kSingleRows && V <= kSingleSlots * vec_elems(dt); }

// Workgroups per long row: one as long as its sixteen wavefronts need few rounds of loads (a join is another launch),
// beyond that enough to occupy the chip.
int parts_of(int64_t rows, int V, int dt) {
  const int64_t rounds = ((int64_t)V + (int64_t)kChunkSlots * vec_elems(dt) - 1) / ((int64_t)kChunkSlots * vec_elems(dt));
  if (rounds <= 16) return 1;
  int64_t parts = (2048 + rows - 1) / rows;
  if (parts > rounds) parts = rounds;
  if (parts > kMaxParts) parts = kMaxParts;
  return parts < 1 ? 1 : (int)parts;
}
// One workgroup to a row that fits its registers (20 slots a thread of 1024).
int64_t row_slots(int V, int dt) { return ((int64_t)V + vec_elems(dt) - 1) / vec_elems(dt); }
bool row_fits(int V, int dt) { return row_slots(V, dt) < 20 * 1024; }

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

template <int DT, int NT>
void launch_fwd_rows_by(const Fwd& a, bool entropy, hipStream_t st) {
  const dim3 grid((unsigned)(a.r.rows * a.parts)), block(NT);
  if (a.top) {
    if (entropy) k_cat_fwd_row<DT, true, true, NT><<<grid, block, 0, st>>>(a);
    else k_cat_fwd_row<DT, false, true, NT><<<grid, block, 0, st>>>(a);
  } else {
    if (entropy) k_cat_fwd_row<DT, true, false, NT><<<grid, block, 0, st>>>(a);
    else k_cat_fwd_row<DT, false, false, NT><<<grid, block, 0, st>>>(a);
  }
}
template <int DT>
void launch_fwd_rows(const Fwd& a, bool entropy, hipStream_t st) {
  if (wide_rows(a.r.rows * a.parts, a.r.V / a.parts, DT)) launch_fwd_rows_by<DT, kWideThreads>(a, entropy, st);
  else if (single_wave_rows(a.r.rows * a.parts, a.r.V / a.parts, DT)) launch_fwd_rows_by<DT, 64>(a, entropy, st);
  else launch_fwd_rows_by<DT, kRowThreads>(a, entropy, st);
}

template <int DT>
void launch_distill_row(const Dist& a, hipStream_t st) {
  // (a row that starts between multiples of 16 bytes may have one slot more)
  const bool aligned = (((uintptr_t)a.r.x | (uintptr_t)(a.r.ld * elem_size(DT))) & 15) == 0;
  const int64_t ns = row_slots(a.r.V, DT) + (aligned ? 0 : 1);
  const dim3 grid((unsigned)a.r.rows);
  // (two wavefronts to the shortest: 16384 x 2500 bfloat16 54 us, by four 69; 20000 x 3000 float32 106 us, by four 94)
  if (ns <= 5 * 128 && a.t.k <= 128) k_cat_distill_row<DT, 128, 5><<<grid, 128, 0, st>>>(a);
  else if (ns <= 2 * 256) k_cat_distill_row<DT, 256, 2><<<grid, 256, 0, st>>>(a);
  else if (ns <= 4 * 256) k_cat_distill_row<DT, 256, 4><<<grid, 256, 0, st>>>(a);
  else if (ns <= 8 * 256) k_cat_distill_row<DT, 256, 8><<<grid, 256, 0, st>>>(a);
  else if (ns <= 16 * 256) k_cat_distill_row<DT, 256, 16><<<grid, 256, 0, st>>>(a);
  else if (ns <= 16 * 512) k_cat_distill_row<DT, 512, 16><<<grid, 512, 0, st>>>(a);
  else if (ns <= 16 * 1024) k_cat_distill_row<DT, 1024, 16><<<grid, 1024, 0, st>>>(a);
  else k_cat_distill_row<DT, 1024, 20><<<grid, 1024, 0, st>>>(a);
}

}  // namespace

extern "C" size_t dmv_cat_log_prob_ws_bytes(const DmvCatRows* r, int32_t top) {
  if (check_rows(r) != DMV_OK || r->rows == 0 || top < 0 || top > kMaxTop || r->V <= kSmallMax) return 0;
  const int parts = parts_of(r->rows, r->V, r->dtype);
  if (parts == 1) return 0;
  return (size_t)r->rows * parts * (sizeof(f32x4) + (size_t)top * sizeof(uint2));
}

extern "C" int dmv_cat_log_prob(const DmvCatRows* r, float* log_prob, float* entropy, int32_t top, float* top_log_prob,
                                int64_t* top_index, float* stats, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check_rows(r);
  if (rc != DMV_OK) return rc;
  if (top < 0) return DMV_E_BADARG;
  if (top > kMaxTop) return DMV_E_UNSUPPORTED;
  if (r->rows == 0) return DMV_OK;
  if ((log_prob && !r->X) || (!log_prob && !entropy && !top) || (top && (!top_log_prob || !top_index))) return DMV_E_BADARG;
  if (((uintptr_t)stats & 15) != 0 || ((uintptr_t)ws & 15) != 0) return DMV_E_BADARG;
  Fwd a{rows_of(r), log_prob, entropy, top, top_log_prob, top_index, (f32x4*)stats, kLog2e, 1, nullptr, nullptr, nullptr, 0};
  hipStream_t st = (hipStream_t)stream;
  if (r->V <= kSmallMax) {
    by_type(r->dtype, [&](auto dt) {
      small_tile<decltype(dt)::value>(r->V, [&](auto t) {
        typedef decltype(t) T;
        const dim3 grid((unsigned)T::groups(r->rows)), block(kSmallThreads);
        auto launch = [&](auto top) {
          constexpr int TOP = decltype(top)::value;
          if (entropy) k_cat_fwd_small<T::DT, T::VEC, T::L, T::SL, true, TOP><<<grid, block, 0, st>>>(a);
          else k_cat_fwd_small<T::DT, T::VEC, T::L, T::SL, false, TOP><<<grid, block, 0, st>>>(a);
        };
        constexpr int parts = T::VEC * T::SL < 8 ? T::VEC * T::SL : 8;      // of a lane's elements, for the bound
        if (!a.top) launch(std::integral_constant<int, kNoTop>());
        else if (2 * a.top <= T::L * parts) launch(std::integral_constant<int, kRanked>());
        else if constexpr (T::L <= 8) launch(std::integral_constant<int, kSorted>());
      });
    });
    DMV_HIP_CHECK_LAUNCH();
    return DMV_OK;
  }
  a.parts = parts_of(r->rows, r->V, r->dtype);
  if (!fits_grid(r->rows * a.parts, single_wave_rows(r->rows, r->V, r->dtype) ? 64 : kRowThreads)) return DMV_E_UNSUPPORTED;
  if (a.parts > 1) {
    if (!ws || ws_bytes < dmv_cat_log_prob_ws_bytes(r, top)) return DMV_E_WORKSPACE;
    a.part = (f32x4*)ws;
    a.part_top = (uint2*)(a.part + r->rows * a.parts);
  }
  by_type(r->dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    launch_fwd_rows<DT>(a, entropy != nullptr, st);
    if (a.parts > 1) k_cat_fwd_join<DT><<<(unsigned)r->rows, kJoinThreads, 0, st>>>(a);
  });
  DMV_HIP_CHECK_LAUNCH();
  return DMV_OK;
}

extern "C" int dmv_cat_log_prob_backward(const DmvCatRows* r, const float* stats, const float* g_log_prob, const float* g_entropy,
                                         int32_t top, const int64_t* top_index, const float* g_top, void* d_logits, int64_t ld_d,
                                         void* stream) {
  const int rc = check_rows(r);
  if (rc != DMV_OK) return rc;
  if (top < 0) return DMV_E_BADARG;
  if (top > kMaxTop) return DMV_E_UNSUPPORTED;
  if (r->rows == 0) return DMV_OK;
  if ((g_log_prob && !r->X) || (g_top && (!top || !top_index)) || ld_d < r->V) return DMV_E_BADARG;
  if (!stats || ((uintptr_t)stats & 15) != 0 || !d_logits || ((uintptr_t)d_logits % elem_size(r->dtype)) != 0) return DMV_E_BADARG;
  Bwd a{rows_of(r), (const f32x4*)stats, g_log_prob, g_entropy, top, top_index, g_top, d_logits, ld_d, 1};
  hipStream_t st = (hipStream_t)stream;
  if (r->V <= kSmallMax) {
    by_type(r->dtype, [&](auto dt) {
      small_tile<decltype(dt)::value>(r->V, [&](auto t) {
        typedef decltype(t) T;
        k_cat_bwd_small<T::DT, T::VEC, T::L, T::SL><<<(unsigned)T::groups(r->rows), kSmallThreads, 0, st>>>(a);
      });
    });
    DMV_HIP_CHECK_LAUNCH();
    return DMV_OK;
  }
  a.chunks = dmv_ceil_div(row_slots(r->V, r->dtype), kChunkSlots);
  if (!fits_grid(r->rows * a.chunks, kRowThreads)) return DMV_E_UNSUPPORTED;
  by_type(r->dtype, [&](auto dt) {
    k_cat_bwd_chunk<decltype(dt)::value><<<(unsigned)(r->rows * a.chunks), kRowThreads, 0, st>>>(a);
  });
  DMV_HIP_CHECK_LAUNCH();
  return DMV_OK;
}

static int check_teacher(const DmvCatRows* r, const DmvCatTeacher* t) {
  if (!t || t->k < 1 || !t->logits || !t->index || t->period < 1 || (t->weight && t->w_period < 1)) return DMV_E_BADARG;
  if (t->dtype < DMV_F32 || t->dtype > DMV_F16 || t->k > kMaxTeacher) return DMV_E_UNSUPPORTED;
  if (((uintptr_t)t->logits % elem_size(t->dtype)) != 0 || !(t->temperature >= 1e-30f && t->temperature <= 1e30f)) return DMV_E_BADARG;
  return DMV_OK;
}
static Dist dist_of(const DmvCatRows* r, const DmvCatTeacher* t) {
  Dist a{};
  a.r = rows_of(r);
  a.r.X = nullptr, a.r.M = nullptr;      // which rows count is said by the weights
  a.t = Teacher{t->logits, t->index, t->weight, t->period, t->w_period, t->k, t->dtype, kLog2e / t->temperature, 1.f / t->temperature};
  a.chunks = a.parts = 1;
  return a;
}
// A small launch: one workgroup does all rows in two rounds at most, and the loss.  A launch less for the host: 16 x 25
// float32 a step of 84 us instead of 93, 64 x 1000 84 instead of 93, each step waited for 100 instead of 108.  On the GPU
// alone, as in a replayed graph, 5.6 us instead of 6.9, and 15.3 instead of 7.6: a third round would lose what it saves.
template <typename T>
bool lone_group(int64_t rows, int k) {
  return rows <= 2 * (kLoneThreads / T::L) && (size_t)(kLoneThreads / T::L) * k * sizeof(Entry) <= 48 * 1024;
}
// shares of the loss that a launch leaves to the sum; 0: it forms the loss itself
static int64_t loss_parts(const DmvCatRows* r, int k) {
  int64_t n = r->rows;
  if (r->V <= kSmallMax)
    by_type(r->dtype, [&](auto dt) {
      teacher_tile<decltype(dt)::value>(r->V, k, [&](auto t) {
        typedef decltype(t) T;
        n = lone_group<T>(r->rows, k) ? 0 : T::groups(r->rows);
      });
    });
  return n;
}

extern "C" size_t dmv_cat_distill_ws_bytes(const DmvCatRows* r, int32_t k) {
  if (check_rows(r) != DMV_OK || r->rows == 0 || k < 1 || k > kMaxTeacher) return 0;
  size_t n = up16((size_t)loss_parts(r, k) * sizeof(double));
  if (r->V > kSmallMax && !row_fits(r->V, r->dtype))
    n += (size_t)r->rows * (1 + parts_of(r->rows, r->V, r->dtype)) * sizeof(f32x4);
  return n;
}

extern "C" int dmv_cat_distill(const DmvCatRows* r, const DmvCatTeacher* t, float* per_row, float* loss, float* stats, void* d_logits,
                               int64_t ld_d, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_rows(r);
  if (rc != DMV_OK) return rc;
  if (!loss || (d_logits && ld_d < r->V)) return DMV_E_BADARG;
  hipStream_t st = (hipStream_t)stream;
  if (r->rows == 0) {
    k_cat_loss<<<1, kLossThreads, 0, st>>>(nullptr, 0, loss);
    DMV_HIP_CHECK_LAUNCH();
    return DMV_OK;
  }
  rc = check_teacher(r, t);
  if (rc != DMV_OK) return rc;
  if (((uintptr_t)stats & 15) != 0 || (d_logits && ((uintptr_t)d_logits % elem_size(r->dtype)) != 0)) return DMV_E_BADARG;
  const size_t need = dmv_cat_distill_ws_bytes(r, t->k);
  if (need && (!ws || ((uintptr_t)ws & 15) != 0 || ws_bytes < need)) return DMV_E_WORKSPACE;
  const int64_t n_loss = loss_parts(r, t->k);
  Dist a = dist_of(r, t);
  a.per_row = per_row;
  a.loss_part = (double*)ws;
  a.stats = (f32x4*)stats;
  a.d = d_logits;
  a.ld_d = ld_d;
  if (r->V <= kSmallMax) {
    by_type(r->dtype, [&](auto dt) {
      teacher_tile<decltype(dt)::value>(r->V, t->k, [&](auto tile) {
        typedef decltype(tile) T;
        if (lone_group<T>(r->rows, t->k)) {
          a.loss = loss;
          const size_t lds = small_lds<T>(t->k) * (kLoneThreads / kSmallThreads);
          k_cat_distill_small<T::DT, T::VEC, T::L, T::SL, kLoneThreads><<<1, kLoneThreads, lds, st>>>(a);
        } else {
          k_cat_distill_small<T::DT, T::VEC, T::L, T::SL, kSmallThreads><<<(unsigned)n_loss, kSmallThreads, small_lds<T>(t->k), st>>>(a);
        }
      });
    });
  } else if (!fits_grid(r->rows, row_slots(r->V, r->dtype) < 5 * 128 && t->k <= 128 ? 128 : kRowThreads)) {
    return DMV_E_UNSUPPORTED;
  } else if (row_fits(r->V, r->dtype)) {
    by_type(r->dtype, [&](auto dt) { launch_distill_row<decltype(dt)::value>(a, st); });
  } else {
    a.parts = parts_of(r->rows, r->V, r->dtype);
    f32x4* own = (f32x4*)((char*)ws + up16((size_t)n_loss * sizeof(double)));
    if (!a.stats) a.stats = own;
    a.part = own + r->rows;
    a.chunks = dmv_ceil_div(row_slots(r->V, r->dtype), kChunkSlots);
    Fwd f{a.r, nullptr, nullptr, 0, nullptr, nullptr, nullptr, a.t.c, a.parts, a.part, nullptr, a.t.weight, a.t.w_period};
    const int64_t items = r->rows * a.chunks;
    by_type(r->dtype, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      launch_fwd_rows<DT>(f, false, st);
      k_cat_distill_join<DT><<<(unsigned)r->rows, kRowThreads, 0, st>>>(a);
      if (a.d) k_cat_distill_chunk<DT><<<(unsigned)(items < 8192 ? items : 8192), kRowThreads, 0, st>>>(a);
    });
  }
  if (!a.loss) k_cat_loss<<<1, kLossThreads, 0, st>>>(a.loss_part, n_loss, loss);
  DMV_HIP_CHECK_LAUNCH();
  return DMV_OK;
}

extern "C" int dmv_cat_distill_backward(const DmvCatRows* r, const DmvCatTeacher* t, const float* gscale, int32_t unless_one,
                                        const float* stats, void* d_logits, int64_t ld_d, void* stream) {
  int rc = check_rows(r);
  if (rc != DMV_OK) return rc;
  if (ld_d < r->V || !gscale) return DMV_E_BADARG;
  if (r->rows == 0) return DMV_OK;
  rc = check_teacher(r, t);
  if (rc != DMV_OK) return rc;
  if (!d_logits || ((uintptr_t)d_logits % elem_size(r->dtype)) != 0) return DMV_E_BADARG;
  if (r->V > kSmallMax && (!stats || ((uintptr_t)stats & 15) != 0)) return DMV_E_BADARG;
  Dist a = dist_of(r, t);
  a.gscale = gscale;
  a.unless_one = unless_one;
  a.stats = r->V > kSmallMax ? (f32x4*)const_cast<float*>(stats) : nullptr;   // short rows form theirs again
  a.d = d_logits;
  a.ld_d = ld_d;
  hipStream_t st = (hipStream_t)stream;
  by_type(r->dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (r->V <= kSmallMax) {
      teacher_tile<DT>(r->V, t->k, [&](auto tile) {
        typedef decltype(tile) T;
        const dim3 grid((unsigned)T::groups(r->rows));
        k_cat_distill_small<T::DT, T::VEC, T::L, T::SL, kSmallThreads><<<grid, kSmallThreads, small_lds<T>(t->k), st>>>(a);
      });
    } else {
      a.chunks = dmv_ceil_div(row_slots(r->V, r->dtype), kChunkSlots);
      const int64_t items = r->rows * a.chunks;
      k_cat_distill_chunk<DT><<<(unsigned)(items < 2048 ? items : 2048), kRowThreads, 0, st>>>(a);
    }
  });
  DMV_HIP_CHECK_LAUNCH();
  return DMV_OK;
}

extern "C" uint64_t dmv_capture_id(void* stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return status == hipStreamCaptureStatusActive ? id : 0;
}
