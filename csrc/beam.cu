// Beam search: the best W continuations of W beams, and the states that follow them.
//
// kf_beam_select.  Of each prompt's W beams with scores s_w and logits l_w (V values each) the W best pairs (w, t) by
//     s_w + l_w[t] - log sum_t' exp(l_w[t']) .
// Within a beam the order of candidates is that of its logits, so W tokens of each beam are all that can be among the best.  One cluster
// of CTAs a prompt; the logits of its beams, one after the other, are dealt out to the CTAs in equal ranges.
//   * One pass over the logits: a thread keeps the largest of its logits and the sum of exp(x - r), with r the largest of its first round; in
//     fp32 over a vector and in 64 bits from there on, because candidates of different beams may lie close together.
//     r moves only when a logit is 8 above it: moved with every new maximum, it cost a branch in most vectors.  The difference is taken
//     before the factor log2 e: large logits lose nothing, and rows of the type's lowest value have exponents of zero like any others.
//   * What a row's sum comes to depends on where the row begins and which threads read it, in the last bits.  So where candidates of different
//     beams are so close that this could decide (NEAR), the first CTA takes these beams' sums again in 64 bits, in the order of the values,
//     and counts places again: equal rows with equal scores tie, whatever their places in memory.
//   * Each of a CTA's 8 warps has ceil(W / 8) threads whose largest logit is at least the warp's ceil(W / 8)-th largest.  So at least W
//     logits reach the least of these over the warps, a bound that costs a warp-wide maximum or a few.  Taken after each thread's first two
//     vectors, and whenever there are twice as many, it leaves about a hundred vectors for 8 beams that reach it and are noted; taken
//     again at the end, about 22.  Lists that every warp kept on the way, with an insertion for each of W ln(n / W) logits, took 98 us for
//     64 x 8 x 128 256 in bf16, reading all vectors of the threads that reach the bound again 92, the notes 40.
//   * Candidates are 64-bit keys: the logit's bits in an order-preserving form, then the complement of its index, so that of equal
//     logits the lowest index is the largest key.  There are few, so a candidate's place is how many are larger, counted; the cluster's
//     CTAs put theirs into the first one's shared memory.
// What bounds it: many prompts, the logits, which are read once (64 x 8 x 128 256 in bf16, an eighth finished: 115 MB in 40 us, 2.9 TB/s: the
// pass at 75 to 80 % of a copy's rate, and behind it, in every CTA at the same time, bounds, candidates and sums); few prompts, these steps
// and the launch (1 x 4 x 32 000: 7.2 us).  Launches are joined to the one before (programmatic launch): by itself a launch of clusters began
// 2.4 us later.
//
// kf_beam_reorder.  state[b, w] = state[b, parent[b, w]] for all states in one launch.  A thread owns 16 bytes of a column: it reads
// the column's W values and then writes them, so that parents may be any selection of beams, also in place, without a second buffer.
// What bounds it: a read and a write of what moves (4 x 8 beams' caches of a 7B model, 1.7 GB: 255 us, 104 % of a copy's rate, since beams
// that keep their place move nothing); small states, the launch and the host's work for it (16 x 8 histories: 5.5 us).
#include "common.cuh"
#include "attention_common.cuh"
#include "decode_common.cuh"

#include <cuda_fp16.h>

namespace kf {
namespace beam {

using namespace kf::attn;   // two-wide arithmetic
using decode::fast_exp2;
using decode::mapa_shared;

constexpr int MAX_BEAMS = 32;   // a warp's list is one key per lane
constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;
// CTAs of a cluster: 16 where all clusters' CTAs have an SM each, which few prompts need (1 x 8 x 128 256: 18.2 -> 13.4 us), else 8.
constexpr int CTAS_FEW = 16, CTAS_MANY = 8;
// Vectors that a CTA reads in the time that bounds and candidates of a second row take it.  Rows dealt out in equal shares / a whole number of
// CTAs each, us: 3 x 5 x 50 257 12.8 / 10.6, 2 x 6 x 128 256 14.7 / 13.5, 2 x 12 x 50 257 18.3 / 15.8, 4 x 7 x 30 000 11.9 / 9.0.
constexpr uint32_t SPARE = 2048;
constexpr int MAX_PARTS = MAX_BEAMS / CTAS_MANY + 1;  // rows that a CTA's range meets
constexpr int NOTES = 512;                            // vectors that a CTA notes (20 KB); more (rising logits, equal ones) go through lists
constexpr int ROOM = 512;                             // candidates that a CTA sorts, likewise

typedef unsigned long long Key;

// The order of floats as unsigned integers (of numbers none is 0); -0 counts as +0.
__device__ __forceinline__ uint32_t ordered(float x) {
  uint32_t u = __float_as_uint(x);
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ Key ordered(double x) {
  Key u = Key(__double_as_longlong(x));
  if (u == 1ull << 63) u = 0;
  return (u >> 63) ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double unordered(Key o) { return __longlong_as_double((long long)((o >> 63) ? o & ~(1ull << 63) : ~o)); }
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ Key make_key(float x, uint32_t index) { return (Key(ordered(x)) << 32) | (0xffffffffu - index); }
__device__ __forceinline__ float key_value(Key k) { return unordered(uint32_t(k >> 32)); }
__device__ __forceinline__ uint32_t key_index(Key k) { return 0xffffffffu - uint32_t(k); }

// Maximum and minimum that keep numbers below the smallest normal one (the build's fast math would make them zeros) and ignore NaN.
__device__ __forceinline__ float max_of(float a, float b) {
  float r;
  asm("max.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_of(float a, float b) {
  float r;
  asm("min.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// e^d for d <= 0, the difference of two references, with an error that does not grow with d: the whole part of d log2 e goes into the
// exponent, and log2 e has 48 bits.  Below -80 is nothing beside a sum of 1.
__device__ __forceinline__ float exp_between(float d) {
  constexpr float LOG2E = 1.4426950408889634f, REST = float(1.4426950408889634 - double(LOG2E));
  d = max_of(d, -80.f);
  const float whole = rintf(__fmul_rn(d, LOG2E)), part = __fmaf_rn(d, REST, __fmaf_rn(d, LOG2E, -whole));
  return __fmul_rn(fast_exp2(part), __int_as_float((int(whole) + 127) << 23));
}

// What the one pass leaves in a logarithm of a sum, at most.  The relative error of a sum is the mean of its terms' errors, which are
//   * of an exponential: 2^-22; of its argument: |d| (2^-24 + 2^-24 + 2^-26), from the difference, the factor and log2 e.  The mean of |d|
//     is at most HIGH + 1 above the reference, and below, with a term next to the reference among n of them, the a - 1 for which
//     a + log(a - 1) = log n + 1/2: 4.3 for 500 of a thread, 11 for the 2^20 that it may have.  So 2.4e-7 + 11 * 1.4e-7;
//   * of the additions: 6 in 32 bits behind a term, 3.6e-7, the rest is in 64;
//   * of exp_between: 2^-22 + 2^-24, at three joins, and with a reference that moves: what has moved three times counts for nothing.
// That is 4e-6 (the most that was seen, over rows made to be so, is 2e-7).  Where candidates of different beams are no further apart than twice as much, the sums are taken again in 64 bits.
constexpr float HIGH = 8.f;   // a reference moves where a logit is this far above it
constexpr double NEAR = 8e-6;

// Key by key: the largest `width` that a warp has met, lane i the i-th (0 = none).
struct TopList {
  Key mine = 0, worst = 0;
  // All lanes call; each offers a key (0 = nothing).
  __device__ __forceinline__ void offer(Key k, int width) {
    const int lane = threadIdx.x & 31;
    uint32_t todo = __ballot_sync(0xffffffffu, k > worst);
    while (todo) {
      const Key in = __shfl_sync(0xffffffffu, k, __ffs(todo) - 1);
      const int place = __popc(__ballot_sync(0xffffffffu, mine > in));
      const Key above = __shfl_up_sync(0xffffffffu, mine, 1);
      if (lane >= place) mine = lane == place ? in : above;
      if (lane >= width) mine = 0;
      worst = __shfl_sync(0xffffffffu, mine, width - 1);
      todo &= todo - 1;
      todo &= __ballot_sync(0xffffffffu, k > worst);
    }
  }
};

// Over eight lanes side by side.
__device__ __forceinline__ int sum_of_8(int x) {
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// 32 bytes of logits, on 32 bytes: the widest load there is.
struct alignas(32) Raw {
  uint32_t w[8];
};
__device__ __forceinline__ Raw load_raw(const Raw* p) {
  Raw v;
  asm("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
      : "l"(p));
  return v;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Them as floats, and their maximum, which is NaN where one of them is.
template <typename T>
struct Logits;
template <>
struct Logits<float> {
  static constexpr uint32_t NONE = 0xff800000u;   // -inf in all of a word
  static constexpr int N = 8;
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ float load(const Raw& v, float (&x)[N]) {
    float m[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(v.w[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = max_or_nan(x[2 * i], x[2 * i + 1]);
    return max_or_nan(max_or_nan(m[0], m[1]), max_or_nan(m[2], m[3]));
  }
};
template <>
struct Logits<__nv_bfloat16> {
  static constexpr uint32_t NONE = 0xff80ff80u;
  static constexpr int N = 16;
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) {
    return __uint_as_float(uint32_t(*reinterpret_cast<const uint16_t*>(p)) << 16);
  }
  static __device__ __forceinline__ float load(const Raw& v, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[2 * i] = __uint_as_float(v.w[i] << 16), x[2 * i + 1] = __uint_as_float(v.w[i] & 0xffff0000u);
    const uint32_t m = max2(max2(max2(v.w[0], v.w[1]), max2(v.w[2], v.w[3])), max2(max2(v.w[4], v.w[5]), max2(v.w[6], v.w[7])));
    return max_or_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
};
template <>
struct Logits<__half> {
  static constexpr uint32_t NONE = 0xfc00fc00u;
  static constexpr int N = 16;
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ float load(const Raw& v, float (&x)[N]) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v.w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
      m = max_or_nan(m, max_or_nan(f.x, f.y));
    }
    return m;
  }
};
// NaN counts as -inf, +inf as the largest number.
__device__ __forceinline__ float clean(float x) { return min_of(max_of(x, -INFINITY), 3.402823466e38f); }

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// e^d for d <= 0 in 64 bits, without a branch, so that several are under way: 2^n e^r with |r| <= log(2) / 2 and the exponential's series up to
// r^12 / 12!, of which r^13 / 13! = 2e-16 is left.  What is below e^-700 counts for nothing beside the 1 of the largest.
__device__ __forceinline__ double exp_below(double d) {
  constexpr double LN2 = 0.6931471805599453, LN2_REST = 2.3190468138462996e-17;   // log 2 in 106 bits
  d = fmax(d, -700.0);
  const double n = rint(d * 1.4426950408889634), r = fma(-n, LN2_REST, fma(-n, LN2, d));
  double y = fma(1.0 / 479001600.0, r, 1.0 / 39916800.0);
  y = fma(y, r, 1.0 / 3628800.0), y = fma(y, r, 1.0 / 362880.0), y = fma(y, r, 1.0 / 40320.0), y = fma(y, r, 1.0 / 5040.0);
  y = fma(y, r, 1.0 / 720.0), y = fma(y, r, 1.0 / 120.0), y = fma(y, r, 1.0 / 24.0), y = fma(y, r, 1.0 / 6.0);
  y = fma(y, r, 0.5), y = fma(y, r, 1.0), y = fma(y, r, 1.0);
  return y * __hiloint2double((1023 + int(n)) << 20, 0);
}

template <typename T>
struct Call {
  const T* logits;
  long long stride_b, stride_w;
  const float* scores;
  const uint8_t* finished;
  int W, V;
  long long eos, pad;
  float* out_scores;
  long long *out_parents, *out_tokens;
  uint8_t* out_finished;
};

// The candidates of a prompt's beams and their places, in shared memory.  The pointers are kept for choose_again: as registers they are spilled.
struct Choice {
  Key* total;                // [W][totals]: scores in the order of integers, best first, 0: none
  uint32_t* token;           // [W][W]
  int totals;
  int winner[MAX_BEAMS];     // of each place: which candidate, beam * MAX_BEAMS + its rank there, or -1
  Key best[MAX_BEAMS];       // its score
  Key next[MAX_BEAMS];       // of each beam: its best candidate without a place, 0: none
};

// A candidate's place: how many come before it, its own beam's better ones, others' better ones, lower beams' equal ones; a warp a beam,
// eight lanes a candidate.
__device__ __forceinline__ void find_places(Choice& c, const Key* total, int totals, int W) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int w = warp; w < W; w += WARPS)
    for (int j0 = 0; j0 < W; j0 += 4) {
      const int j = j0 + lane / 8;
      const Key mine = j < W ? total[w * totals + j] : 0;
      int before = 0;
      for (int x = lane & 7; x < W; x += 8) {
        const Key* of = total + x * totals;
        const Key limit = mine - (x < w);
        int n = 0;
        for (int k = 0; k < W; k += 8)   // zeros behind the last one
#pragma unroll
          for (int e = 0; e < 8; ++e) n += of[k + e] > limit;
        before += x == w ? j : n;
      }
      before = sum_of_8(before);
      const bool among = mine && before < W;
      const bool ahead = __shfl_up_sync(0xffffffffu, int(among), 8) || lane < 8;   // the one before it has a place
      if ((lane & 7) == 0 && mine) {
        if (among) c.winner[before] = w * MAX_BEAMS + j, c.best[before] = mine;
        else if (ahead) c.next[w] = mine;
      }
      if (!__all_sync(0xffffffffu, among)) break;   // nor are those behind
    }
}

template <typename T>
__device__ __forceinline__ void write_places(const Call<T>& a, const Choice& c, const uint32_t* token, long long first, uint32_t ends, int W) {
  const int tid = threadIdx.x;
  if (tid >= W) return;
  const int i = c.winner[tid], parent = i < 0 ? tid : i / MAX_BEAMS;
  const bool ended = i >= 0 && ((ends >> parent) & 1u);
  const long long t = i < 0 || ended ? a.pad : (long long)token[parent * W + i % MAX_BEAMS];
  a.out_scores[first + tid] = i < 0 ? -INFINITY : float(unordered(c.best[tid]));
  a.out_parents[first + tid] = parent;
  a.out_tokens[first + tid] = t;
  a.out_finished[first + tid] = ended || (i >= 0 && t == a.eos);
}

// Places once more, with the scores of some beams (`near`, those of `live` among them with logits) from sums in 64 bits: value i by thread
// i % THREADS, so that equal rows have equal sums wherever they lie.  Where all rows are equal one sum will do, whatever its last bits.
// Nothing follows this, so that the pass keeps no registers for it; that, and not a call (0.1 to 0.5 us for every selection).
template <typename T>
__device__ __forceinline__ void choose_again(const Call<T>& a, Choice& c, long long b, uint32_t near, uint32_t live, uint32_t ends,
                                             double* of_warps) {
  constexpr int AT_ONCE = 8;
  const int tid = threadIdx.x, W = a.W;
  const int lead = __ffs(near & live) - 1;
  const T* x0 = a.logits + b * a.stride_b + lead * a.stride_w;
  int same = (near & ~live) == 0;
  for (uint32_t left = near & live & ~(1u << lead); same && left; left &= left - 1) {
    const T* x = a.logits + b * a.stride_b + (__ffs(left) - 1) * a.stride_w;
#pragma unroll 1
    for (int i0 = tid; i0 < a.V; i0 += AT_ONCE * THREADS)
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e)
        if (i0 + e * THREADS < a.V) same &= clean(Logits<T>::one(x + i0 + e * THREADS)) == clean(Logits<T>::one(x0 + i0 + e * THREADS));
    same = __syncthreads_and(same);
  }
  double lse = clean(Logits<T>::one(x0 + c.token[lead * W])) - (unordered(c.total[lead * c.totals]) - double(a.scores[b * W + lead]));
  __syncthreads();   // the total has been read
  for (uint32_t left = near & live; left; left &= left - 1) {
    const int w = __ffs(left) - 1;
    const T* x = a.logits + b * a.stride_b + w * a.stride_w;
    if (!same) {
      const double top = clean(Logits<T>::one(x + c.token[w * W]));
      double sum = 0.0;
#pragma unroll 1
      for (int i0 = tid; i0 < a.V; i0 += AT_ONCE * THREADS) {
        float v[AT_ONCE];
#pragma unroll
        for (int e = 0; e < AT_ONCE; ++e) v[e] = i0 + e * THREADS < a.V ? clean(Logits<T>::one(x + i0 + e * THREADS)) : -INFINITY;
#pragma unroll
        for (int e = 0; e < AT_ONCE; ++e) sum += exp_below(double(v[e]) - top);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if ((tid & 31) == 0) of_warps[tid >> 5] = sum;
      __syncthreads();
      sum = of_warps[0];
      for (int i = 1; i < WARPS; ++i) sum += of_warps[i];
      lse = top + log(sum);
    }
    Key* mine = c.total + w * c.totals + tid;
    if (tid < W && *mine) *mine = ordered(double(a.scores[b * W + w]) + (double(clean(Logits<T>::one(x + c.token[w * W + tid]))) - lse));
    __syncthreads();   // of_warps has been read
  }
  find_places(c, c.total, c.totals, W);
  __syncthreads();
  write_places(a, c, c.token, b * W, ends, W);
}

// Four CTAs an SM, which is 64 registers: with logits of 16 bits 80 bytes are spilled and 130 read back.  With three and none, us:
// 1 x 8 x 128 256 13.4 / 12.8, 40 x 8 x 50 257 22.3 / 18.0, but 64 x 8 x 128 256 40.1 / 49.2, 64 x 8 x 32 000 in fp32 21.9 / 27.7.
template <typename T>
__global__ void __launch_bounds__(THREADS, 4)
kf_beam_select(const __grid_constant__ Call<T> a) {
  constexpr int N = Logits<T>::N;
  constexpr float LOG2E = 1.4426950408889634f;
  constexpr int UNROLL = 2;
  // What a CTA found in its part of a row, in the first CTA's memory.  Part (nth row, CTA) has number nth + CTA: along the vectors every
  // step raises one of the two.
  struct Part {
    double r, sum;
    Key keys[MAX_BEAMS];
  };
  __shared__ Part parts[MAX_BEAMS + CTAS_FEW];
  __shared__ float rs[2][WARPS];
  __shared__ double sums[2][WARPS];
  __shared__ uint32_t reach[2][WARPS];             // after the first round, at the end
  __shared__ int n_found[MAX_PARTS], n_notes[MAX_PARTS];
  __shared__ Key notes[NOTES];                     // (largest logit, vector)
  __shared__ Raw noted_raw[NOTES];                 // the vector
  __shared__ Key found[ROOM];                      // candidates, or the warps' lists; later the candidates' tokens
  __shared__ Choice choice;
  __shared__ uint32_t again;                       // beams that choose_again looks at
  const int W = a.W, V = a.V;
  Key* total = reinterpret_cast<Key*>(noted_raw);
  const int totals = (W + 7) / 8 * 8 + 1;          // an odd number spreads the beams' over the banks
  uint32_t* token = reinterpret_cast<uint32_t*>(found);
  static_assert(sizeof(noted_raw) >= MAX_BEAMS * (MAX_BEAMS + 1) * sizeof(Key) && alignof(Raw) >= alignof(Key) &&
                    sizeof(found) >= MAX_BEAMS * MAX_BEAMS * sizeof(uint32_t) && alignof(Key) >= alignof(uint32_t),
                "what `total` and `token` lie in");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const uint32_t ctas = cluster_nctaid();
  const int rank = int(cluster_ctarank());
  const long long b = blockIdx.x / ctas, first = b * W;
  if (tid < MAX_PARTS) n_found[tid] = n_notes[tid] = 0;
  if (tid < MAX_BEAMS) choice.winner[tid] = -1, choice.next[tid] = 0;
  if (tid == 0) choice.total = total, choice.token = token, choice.totals = totals;
  grid_dep_wait();
  grid_dep_launch();
  // No pointer is __restrict__: loads of what it says is constant may move ahead of the wait.
  // Beams whose logits count.  One without a score above -inf (or with NaN) has no candidates, a finished one has itself.
  const float score = lane < W ? a.scores[first + lane] : -INFINITY;
  const bool alive = score > -INFINITY;
  const bool done = lane < W && a.finished != nullptr && a.finished[first + lane];
  const uint32_t live = __ballot_sync(0xffffffffu, alive && !done);
  // vectors of a row, at most, so that CTAs meet eighths of rows
  uint32_t per = (max(1u, uint32_t(V) / N) + CTAS_FEW - 1) / CTAS_FEW * CTAS_FEW;
  const uint32_t lives = __popc(live);
  uint32_t chunk = lives * per / ctas;
  if (ctas == CTAS_FEW && lives > 2 && lives <= CTAS_FEW) {   // few prompts: no CTA with parts of two rows, if that is no more than SPARE more
    const uint32_t ways = CTAS_FEW / lives, each = (per + ways - 1) / ways;
    if (each <= chunk + SPARE) chunk = each, per = each * ways;
  }
  const uint32_t r1 = min(chunk * (rank + 1), lives * per);
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // waited for below: the first CTA is there to be written to

  int part = 0;
  for (uint32_t pos = chunk * rank; pos < r1; ++part) {
    const uint32_t nth = pos / per;
    const int v0 = int(pos - nth * per), v_end = int(min(r1 - pos, per - v0)) + v0;
    pos += v_end - v0;
    // the nth live beam
    const int w = __ffs(__ballot_sync(0xffffffffu, ((live >> lane) & 1u) && __popc(live & ((1u << lane) - 1u)) == int(nth))) - 1;
    const T* x0 = a.logits + b * a.stride_b + w * a.stride_w;
    // vectors from the row's first 32-byte boundary on; what is left at both ends goes with the first vector, a value a thread
    const int misaligned = int(reinterpret_cast<uintptr_t>(x0) & 31) / int(sizeof(T));
    const int head = misaligned ? min(V, N - misaligned) : 0;
    const int vectors = (V - head) / N, tail0 = head + vectors * N;
    const int v1 = min(v_end, vectors);
    const Raw* vec = reinterpret_cast<const Raw*>(x0 + head);
    const int single = v0 != 0 || tid >= 2 * N ? -1 : tid < head ? tid : tid >= N && tid - N < V - tail0 ? tail0 + tid - N : -1;
    // Rounds of a vector a thread: two streams, the whole rounds' first and second half, and a last turn with what is left; a vector is
    // asked for as the one before it is taken.
    const int n_vec = v1 > v0 ? v1 - v0 : 0, half = n_vec / THREADS / UNROLL;
    const Raw* mine0 = vec + v0 + tid;
    auto round_of = [&](int u, int j) { return j < half ? u * half + j : UNROLL * half + u; };
    auto fetch = [&](int u, int j) {
      if (j < half) return load_raw(mine0 + (u * half + j) * THREADS);
      Raw v;   // vectors that are not there hold -inf
#pragma unroll
      for (int e = 0; e < 8; ++e) v.w[e] = Logits<T>::NONE;
      if (j == half && (UNROLL * half + u) * THREADS + tid < n_vec) v = load_raw(mine0 + (UNROLL * half + u) * THREADS);
      return v;
    };
    Raw now[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) now[u] = fetch(u, 0);
    const float alone = single >= 0 ? clean(Logits<T>::one(x0 + single)) : -INFINITY;

    // ---- the first round's largest
    float m = alone;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float x[N];
      float mx = Logits<T>::load(now[u], x);
      if (!(mx < INFINITY)) {
        mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < N; ++j) mx = max_of(mx, clean(x[j]));
      }
      m = max_of(m, mx);
    }
    // what ceil(W / warps) of the warp's threads reach, of `full` warps that have a vector a thread (0: fewer have a logit)
    const int full = max(1, min(WARPS, (v1 - v0) / 32));
    auto reached = [&]() {
      uint32_t left = m > -INFINITY ? ordered(m) : 0u, top = __reduce_max_sync(0xffffffffu, left);
      for (int i = full; i < W; i += full) {   // the next largest: one thread less each time
        if (lane == __ffs(__ballot_sync(0xffffffffu, left == top)) - 1) left = 0u;
        top = __reduce_max_sync(0xffffffffu, left);
      }
      return top;
    };
    auto least_of = [&](const uint32_t (&of)[WARPS]) {
      uint32_t least = of[0];
      for (int i = 1; i < full; ++i) least = min(least, of[i]);
      return least;
    };
    volatile uint32_t* so_far = reach[0];
    auto publish = [&]() {
      const uint32_t top = reached();
      if (lane == 0) so_far[warp] = top;
    };
    float least_f = -INFINITY;
    auto bound = [&]() {   // what a warp reaches only grows: an older value of another one is a bound as well
      uint32_t least = so_far[0];
      for (int i = 1; i < full; ++i) least = min(least, so_far[i]);
      if (least) least_f = unordered(least);
    };
    publish();
    __syncthreads();
    bound();

    // ---- the pass: exp(x - r); limit: the logit that is HIGH above r
    // Whole numbers, so that differences of references are exact (those beyond 2^24 differ by nothing, or by so much that it does not matter).
    float r = m > -INFINITY ? rintf(m) : 0.f, limit = m > -INFINITY ? r + HIGH : -INFINITY;
    float usual = fminf(least_f, limit);   // vectors whose largest is below only add to the sum
    double sum = alone > -INFINITY ? double(fast_exp2((alone - r) * LOG2E)) : 0.0;
#pragma unroll 1
    for (int j = 0; j <= half; ++j) {
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        float x[N];
        float mx = Logits<T>::load(now[u], x);
        if (!(mx < usual)) {
          if (!(mx < INFINITY)) {
            mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < N; ++e) mx = max_of(mx, x[e] = clean(x[e]));
          }
          if (mx > limit) {
            const float to = rintf(mx);
            if (limit > -INFINITY) sum *= double(exp_between(r - to));
            r = to;
            limit = r + HIGH;
          }
          if (mx >= least_f && mx > -INFINITY) {
            const int to = atomicAdd(&n_notes[part], 1);
            if (to < NOTES) notes[to] = make_key(mx, uint32_t(v0 + round_of(u, j) * THREADS + tid)), noted_raw[to] = now[u];
          }
          usual = fminf(least_f, limit);
        }
        now[u] = fetch(u, j + 1);
        m = max_of(m, mx);
        const uint64_t r2 = pack2(-r, -r), log2e2 = pack2(LOG2E, LOG2E);
        uint64_t sum2[2];   // of the vector: 32 bits take few terms, and 64 what they come to
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          float y0, y1;
          unpack2(fmul2(fadd2(pack2(x[e], x[e + 1]), r2), log2e2), y0, y1);
          const uint64_t terms = pack2(fast_exp2(y0), fast_exp2(y1));
          sum2[(e >> 1) & 1] = e < 4 ? terms : fadd2(sum2[(e >> 1) & 1], terms);
        }
        float even, odd;
        unpack2(fadd2(sum2[0], sum2[1]), even, odd);
        sum += double(even + odd);
      }
      if (j > 0 && (j & (j - 1)) == 0) {   // of twice as many vectors
        publish();
        __syncwarp();
        bound();
        usual = fminf(least_f, limit);
      }
    }

    // ---- the warp's sum, and the bound again
    {
      const float own_r = m > -INFINITY ? r : -INFINITY;
      float wr = own_r;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) wr = max_of(wr, __shfl_xor_sync(0xffffffffu, wr, o));
      double ws = m > -INFINITY ? sum * double(exp_between(own_r - wr)) : 0.0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
      const uint32_t top = reached();
      if (lane == 0) rs[part & 1][warp] = wr, sums[part & 1][warp] = ws, reach[1][warp] = top;
    }
    __syncthreads();
    const uint32_t least = least_of(reach[1]);
    // ---- the noted vectors that reach it
    auto take = [&](float x, int i) {
      if (x > -INFINITY && ordered(x) >= least) {
        const int to = atomicAdd(&n_found[part], 1);
        if (to < ROOM) found[to] = make_key(x, uint32_t(i));
      }
    };
    const int noted = n_notes[part];
    const float reached_f = least ? unordered(least) : -INFINITY;
    take(alone, single);
    for (int e = tid; e < min(noted, NOTES); e += THREADS) {
      const Key n = notes[e];
      if (uint32_t(n >> 32) >= least) {
        const int at = head + int(key_index(n)) * N;
        float x[N];
        Logits<T>::load(noted_raw[e], x);
        uint32_t hits = 0;   // as floats: those below the smallest normal number are all alike, and looked at again
#pragma unroll
        for (int j = 0; j < N; ++j) hits |= uint32_t(!(clean(x[j]) < reached_f)) << j;
        for (; hits; hits &= hits - 1) {
          const int j = __ffs(hits) - 1;
          take(clean(Logits<T>::one(reinterpret_cast<const T*>(&noted_raw[e]) + j)), at + j);
        }
      }
    }
    __syncthreads();
    // ---- the W largest and the sum, into the first CTA
    if (part == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    const uint32_t to = mapa_shared(smem_u32(&parts[nth + rank]), 0);
    const int candidates = n_found[part];
    if (candidates <= ROOM && noted <= NOTES) {
      if (tid < W && tid >= candidates) st_cluster_u64(to + 16 + 8 * tid, 0ull);
      for (int e0 = warp * 4; e0 < candidates; e0 += WARPS * 4) {   // eight lanes a candidate
        const int e = e0 + lane / 8;
        const Key mine = found[min(e, candidates - 1)];
        int larger = 0;
#pragma unroll 4
        for (int i = lane & 7; i < candidates; i += 8) larger += found[i] > mine;
        larger = sum_of_8(larger);
        if ((lane & 7) == 0 && e < candidates && larger < W) st_cluster_u64(to + 16 + 8 * larger, mine);
      }
    } else {
      // rising or equal logits: every warp through the whole of its vectors
      TopList list;
      for (int base = v0 + warp * 32; base < v1; base += THREADS) {
        const int i = base + lane;
        float x[N], mx = -INFINITY;
        if (i < v1) Logits<T>::load(load_raw(vec + i), x);
#pragma unroll
        for (int j = 0; j < N; ++j) mx = max_of(mx, x[j] = i < v1 ? clean(x[j]) : -INFINITY);
        if (!__any_sync(0xffffffffu, mx > -INFINITY && ordered(mx) >= max(least, uint32_t(list.worst >> 32)))) continue;
#pragma unroll 1
        for (int j = 0; j < N; ++j) list.offer(x[j] > -INFINITY ? make_key(x[j], uint32_t(head + i * N + j)) : 0, W);
      }
      if (warp == 0) list.offer(alone > -INFINITY ? make_key(alone, uint32_t(single)) : 0, W);
      found[warp * MAX_BEAMS + lane] = list.mine;
      __syncthreads();
      if (warp == 0) {
        for (int i = 1; i < WARPS; ++i) list.offer(found[i * MAX_BEAMS + lane], W);
        if (lane < W) st_cluster_u64(to + 16 + 8 * lane, list.mine);
      }
    }
    if (warp == WARPS - 1) {   // it has the fewest candidates
      const float own = lane < WARPS ? rs[part & 1][lane] : -INFINITY;
      float pr = own;
#pragma unroll
      for (int o = WARPS / 2; o > 0; o >>= 1) pr = max_of(pr, __shfl_xor_sync(0xffffffffu, pr, o));
      double ps = own > -INFINITY ? sums[part & 1][lane] * double(exp_between(own - pr)) : 0.0;
#pragma unroll
      for (int o = WARPS / 2; o > 0; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
      if (lane == 0) {
        st_cluster_u64(to, (unsigned long long)__double_as_longlong(double(pr)));
        st_cluster_u64(to + 8, (unsigned long long)__double_as_longlong(ps));
      }
    }
  }

  if (part == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");   // this CTA had nothing to write
  cluster_sync_all();
  // ---- the first CTA joins what the cluster found, a warp a beam
  if (rank != 0) return;
  const double NONE = -INFINITY;
  for (int w = warp; w < W; w += WARPS) {
    const double own_score = double(__shfl_sync(0xffffffffu, score, w));
    if (lane < totals - 1) total[w * totals + lane] = 0;
    __syncwarp();
    if ((live >> w) & 1u) {
      const uint32_t nth = uint32_t(__popc(live & ((1u << w) - 1u)));
      const int c0 = int(nth * per / chunk), count = int((nth * per + per - 1) / chunk) - c0 + 1;   // CTAs that hold its vectors
      const Part* p = parts + nth + c0;
      const double own_r = lane < count ? p[lane].r : NONE;
      double r = own_r;
#pragma unroll
      for (int o = CTAS_FEW / 2; o > 0; o >>= 1) r = fmax(r, __shfl_xor_sync(0xffffffffu, r, o));
      double sum = own_r > NONE ? p[lane].sum * double(exp_between(float(own_r - r))) : 0.0;
#pragma unroll
      for (int o = CTAS_FEW / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const double lse = __shfl_sync(0xffffffffu, r + log(sum), 0);
      for (int i = lane; i < count * W; i += 32) {
        const Key mine = p[i / W].keys[i % W];
        int larger = 0;
        for (int c = 0; c < count; ++c)
          for (int j = 0; j < W; ++j) larger += p[c].keys[j] > mine;
        if (mine && larger < W) {
          total[w * totals + larger] = ordered(own_score + (double(key_value(mine)) - lse));
          token[w * W + larger] = key_index(mine);
        }
      }
    } else if (lane == 0 && own_score > NONE) {
      total[w * totals] = ordered(own_score);   // finished
    }
  }
  __syncthreads();
  const uint32_t ends = __ballot_sync(0xffffffffu, done);
  find_places(choice, total, totals, W);
  __syncthreads();
  write_places(a, choice, token, first, ends, W);
  // ---- meanwhile: candidates of different beams that may have changed places, neighbours that are NEAR, the last one and any beam's next
  if (warp == 1) {
    const int parent = lane < W ? choice.winner[lane] >> 5 : -1, above_parent = lane > 0 && lane < W ? choice.winner[lane - 1] >> 5 : -1;
    const int last_parent = choice.winner[W - 1] >> 5;
    uint32_t beams = 0;
    if (parent >= 0 && above_parent >= 0 && parent != above_parent && unordered(choice.best[lane - 1]) - unordered(choice.best[lane]) <= NEAR)
      beams = 1u << parent | 1u << above_parent;
    const Key behind = choice.next[lane];
    if (behind && last_parent >= 0 && lane != last_parent && unordered(choice.best[W - 1]) - unordered(behind) <= NEAR)
      beams |= 1u << lane | 1u << last_parent;
    beams = __reduce_or_sync(0xffffffffu, beams);
    if (lane == 0) again = beams & live ? beams : 0u;
  }
  __syncthreads();
  if (again) choose_again(a, choice, b, again, live, ends, sums[0]);
}

template <typename T>
static int launch_select(const Call<T>& call, int B, int num_sms, cudaStream_t stream) {
  auto kern = kf_beam_select<T>;
  static bool attr_set[16] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 16 || !attr_set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return 300 + (int)e;
    if (dev < 16) attr_set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  const int ctas = (long long)B * CTAS_FEW <= num_sms ? CTAS_FEW : CTAS_MANY;
  if ((long long)B * ctas > 0x7fffffffLL) return 6;
  cfg.gridDim = dim3((unsigned)(B * ctas));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, call);
  return e == cudaSuccess ? 0 : 500 + (int)e;
}

// ------------------------------------------------------------------ reorder
struct State {
  const uint8_t* src;
  uint8_t* dst;
  long long src_b, src_w, dst_b, dst_w;   // bytes
  long long bytes;                        // of a beam that follow it
};
constexpr int MAX_STATES = 60;            // with the rest of the arguments below 4 KB
struct States {
  State s[MAX_STATES];
};

// T: the widest word that all addresses and steps are multiples of.  A column is one word of all W beams; the last column of a state may
// hold fewer bytes than a word and is moved byte by byte.  Block (x, prompt, state); a thread moves COLS columns, whose words are all
// under way at once: W * COLS of 16 bytes are what fills a GPU's memory with threads enough.
template <typename T, int W, int COLS>
__global__ void __launch_bounds__(256)
kf_beam_reorder(const __grid_constant__ States st, int beams, const void* parents, int wide) {
  grid_dep_wait();
  grid_dep_launch();
  const State& a = st.s[blockIdx.z];
  const long long b = blockIdx.y;
  const long long off0 = ((long long)blockIdx.x * (256 * COLS) + threadIdx.x) * (long long)sizeof(T);
  if ((long long)blockIdx.x * (256 * COLS) * (long long)sizeof(T) >= a.bytes) return;
  const uint8_t* src = a.src + b * a.src_b;
  uint8_t* dst = a.dst + b * a.dst_b;
  int from[W];   // a parent that is no beam, or in place the beam itself: it stays as it is (-1)
#pragma unroll
  for (int w = 0; w < W; ++w) {
    from[w] = -1;
    if (w < beams) {
      const long long at = b * beams + w;
      const long long p = wide ? reinterpret_cast<const long long*>(parents)[at] : (long long)reinterpret_cast<const int*>(parents)[at];
      if (p >= 0 && p < beams && !(a.src == a.dst && p == w)) from[w] = int(p);
    }
  }
  T v[COLS][W];
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    const long long off = off0 + c * 256 * (long long)sizeof(T), left = a.bytes - off;
    if (left >= (long long)sizeof(T)) {
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (from[w] >= 0) v[c][w] = *reinterpret_cast<const T*>(src + from[w] * a.src_w + off);
    }
  }
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    const long long off = off0 + c * 256 * (long long)sizeof(T), left = a.bytes - off;
    if (left >= (long long)sizeof(T)) {
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (from[w] >= 0) *reinterpret_cast<T*>(dst + w * a.dst_w + off) = v[c][w];
    } else if (left > 0) {
      for (int j = 0; j < int(left); ++j) {   // a byte of all beams at a time
        uint8_t byte[W];
#pragma unroll
        for (int w = 0; w < W; ++w)
          if (from[w] >= 0) byte[w] = src[from[w] * a.src_w + off + j];
#pragma unroll
        for (int w = 0; w < W; ++w)
          if (from[w] >= 0) dst[w * a.dst_w + off + j] = byte[w];
      }
    }
  }
}

template <typename T, int W, int COLS>
static void launch_columns(const States& st, int n, int B, int beams, const void* parents, int wide, long long bytes, cudaStream_t stream) {
  const long long step = 256LL * COLS * sizeof(T);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((bytes + step - 1) / step), (unsigned)B, (unsigned)n);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kf_beam_reorder<T, W, COLS>, st, beams, parents, wide);   // the caller asks for the last error
}

template <typename T>
static void launch_reorder(const States& st, int n, int B, int beams, const void* parents, int wide, long long bytes, cudaStream_t stream) {
  if (beams <= 4) launch_columns<T, 4, 2>(st, n, B, beams, parents, wide, bytes, stream);
  else if (beams <= 8) launch_columns<T, 8, 1>(st, n, B, beams, parents, wide, bytes, stream);
  else if (beams <= 16) launch_columns<T, 16, 1>(st, n, B, beams, parents, wide, bytes, stream);
  else launch_columns<T, 32, 1>(st, n, B, beams, parents, wide, bytes, stream);
}

}  // namespace beam
}  // namespace kf

extern "C" {

// logits (B, W, V) with strides in elements and V side by side; type 0 bf16, 1 fp32, 2 fp16.  scores (B, W) fp32, finished (B, W) bytes
// or null.  Writes scores, parents, tokens and finished (B, W).
int kf_beam_select(const void* logits, int type, long long stride_b, long long stride_w, const void* scores, const void* finished, int B, int W,
                   int V, long long eos, long long pad, void* out_scores, void* out_parents, void* out_tokens, void* out_finished, int num_sms,
                   void* stream) {
  using namespace kf::beam;
  if (B < 1 || W < 1 || W > MAX_BEAMS || V < 1 || V > 1 << 28) return 3;   // vectors of 32 rows are counted in 32 bits
  auto go = [&](auto first) {
    using T = decltype(first);
    const Call<T> call{(const T*)logits, stride_b, stride_w, (const float*)scores, (const uint8_t*)finished, W, V, eos, pad, (float*)out_scores,
                       (long long*)out_parents, (long long*)out_tokens, (uint8_t*)out_finished};
    return launch_select(call, B, num_sms, (cudaStream_t)stream);
  };
  if (type == 0) return go(__nv_bfloat16());
  if (type == 1) return go(float());
  if (type == 2) return go(__half());
  return 4;
}

int kf_beam_max_states() { return kf::beam::MAX_STATES; }

// table: 7 numbers a state (src, dst, and in bytes: steps of src and dst from prompt to prompt and beam to beam as src_b, src_w, dst_b,
// dst_w, and the length that moves).  parents (B, beams), int64 or (wide == 0) int32.  dst is src itself or does not overlap it.
int kf_beam_reorder(const long long* table, int n, int B, int beams, const void* parents, int wide, void* stream) {
  using namespace kf::beam;
  if (n < 1 || n > MAX_STATES || B < 1 || B > 65535 || beams < 1 || beams > MAX_BEAMS) return 3;
  States st;
  unsigned long long all = 0;
  long long most = 0;
  for (int i = 0; i < n; ++i) {
    const long long* t = table + 7 * i;
    st.s[i] = State{(const uint8_t*)t[0], (uint8_t*)t[1], t[2], t[3], t[4], t[5], t[6]};
    if (t[6] < 0) return 3;
    if (t[6] > most) most = t[6];
    for (int j = 0; j < 6; ++j) all |= (unsigned long long)t[j];
  }
  if (most == 0) return 0;
  if (most > 1LL << 37) return 6;   // blocks of 256 bytes are counted in 31 bits
  cudaStream_t s = (cudaStream_t)stream;
  if (!(all & 15)) launch_reorder<uint4>(st, n, B, beams, parents, wide, most, s);
  else if (!(all & 7)) launch_reorder<unsigned long long>(st, n, B, beams, parents, wide, most, s);
  else if (!(all & 3)) launch_reorder<uint32_t>(st, n, B, beams, parents, wide, most, s);
  else if (!(all & 1)) launch_reorder<uint16_t>(st, n, B, beams, parents, wide, most, s);
  else launch_reorder<uint8_t>(st, n, B, beams, parents, wide, most, s);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + (int)e;
}

}  // extern "C"
