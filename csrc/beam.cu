// Beam search: the best W continuations of W beams, and the states that follow them.
//
// kf_beam_select.  Of each prompt's W beams with scores s_w and logits l_w (V values each) the W best pairs (w, t) by
//     s_w + l_w[t] - log sum_t' exp(l_w[t']) .
// Within a beam the order of candidates is that of its logits, so W tokens of each beam are all that can be among the best.  One cluster
// of CTAs a prompt; the logits of its beams, one after the other, are dealt out to the CTAs in equal ranges.
//   * One pass over the logits: a thread keeps the largest of its logits and the sum of exp(x - largest), in fp32 over at most a few hundred
//     terms and in 64 bits from there on, because candidates of different beams may lie close together.  The difference is taken before the
//     factor log2 e: rows of the type's lowest value have exponents of zero like any others, and no product overflows.
//   * The W-th largest of the threads' largest logits is at most the W-th largest logit, so only threads whose largest is not below it
//     can hold one of the W best: about W of them, whose logits are read again (out of L2).  A list that every warp kept on the way, which
//     costs an insertion for each of W ln(n / W) logits, took 98 us where this takes 24 (64 x 8 x 128 256 bf16).
//   * Candidates are 64-bit keys: the logit's bits in an order-preserving form, then the complement of its index, so that of equal
//     logits the lowest index is the largest key; sorted by a warp, and joined over the cluster through distributed shared memory.
// What bounds it: the logits are read once.
//
// kf_beam_reorder.  state[b, w] = state[b, parent[b, w]] for all states in one launch.  A thread owns 16 bytes of a column: it reads
// the column's W values and then writes them, so that parents may be any selection of beams, also in place, without a second buffer.
#include "common.cuh"
#include "decode_common.cuh"

#include <cuda_fp16.h>

namespace kf {
namespace beam {

using decode::mapa_shared;

constexpr int MAX_BEAMS = 32;   // a warp's list is one key per lane
constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;
constexpr int MIN_CTAS = 8;     // of a cluster
constexpr int MAX_PARTS = MAX_BEAMS / MIN_CTAS + 1;   // rows that a CTA's range meets
constexpr int ROOM = WARPS * MAX_BEAMS;       // candidates that a CTA sorts; more (equal logits) go through lists
constexpr double LOG2E_D = 1.44269504088896340736;

typedef unsigned long long Key;

// The order of floats as unsigned integers; -0 counts as +0.
__device__ __forceinline__ uint32_t ordered(float x) {
  uint32_t u = __float_as_uint(x);
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ Key make_key(float x, uint32_t index) { return (Key(ordered(x)) << 32) | (0xffffffffu - index); }
__device__ __forceinline__ float key_value(Key k) { return unordered(uint32_t(k >> 32)); }
__device__ __forceinline__ uint32_t key_index(Key k) { return 0xffffffffu - uint32_t(k); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

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

// One step of a warp's sorting network: lanes `j` apart, the larger one to the lower lane where `down`.
template <typename K>
__device__ __forceinline__ K exchange(K k, int j, bool down) {
  const K other = __shfl_xor_sync(0xffffffffu, k, j);
  const bool larger = ((threadIdx.x & j) == 0) == down;
  return (k > other) == larger ? k : other;
}
// A warp's keys, largest first.
template <typename K>
__device__ __forceinline__ K sorted(K k) {
#pragma unroll
  for (int n = 2; n <= 32; n *= 2)
#pragma unroll
    for (int j = n / 2; j > 0; j /= 2) k = exchange(k, j, (threadIdx.x & n & 31) == 0);
  return k;
}
// The 32 largest of two sorted lists.
__device__ __forceinline__ Key merged(Key a, Key b) {
  const Key other = __shfl_sync(0xffffffffu, b, 31 - (threadIdx.x & 31));
  Key k = a > other ? a : other;
#pragma unroll
  for (int j = 16; j > 0; j /= 2) k = exchange(k, j, true);
  return k;
}

// Logits as floats: 16 bytes of them.  NaN counts as -inf, +inf as the type's largest number.
template <typename T>
struct Logits;
template <>
struct Logits<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float clean(float x) { return min_of(max_of(x, -INFINITY), 3.402823466e38f); }
  static __device__ __forceinline__ void load(const uint4& v, float (&x)[N]) {
    x[0] = clean(__uint_as_float(v.x)), x[1] = clean(__uint_as_float(v.y)), x[2] = clean(__uint_as_float(v.z)), x[3] = clean(__uint_as_float(v.w));
  }
  static __device__ __forceinline__ float one(const float* p) { return clean(*p); }
};
template <>
struct Logits<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ uint32_t clean2(uint32_t u) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0xff80ff80u));
    asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(r), "r"(0x7f7f7f7fu));
    return r;
  }
  static __device__ __forceinline__ void load(const uint4& v, float (&x)[N]) {
    const uint32_t u[4] = {clean2(v.x), clean2(v.y), clean2(v.z), clean2(v.w)};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(u[i] << 16), x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) {
    return __uint_as_float(clean2(uint32_t(*reinterpret_cast<const uint16_t*>(p))) << 16);
  }
};
template <>
struct Logits<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), 65504.f); }
  static __device__ __forceinline__ void load(const uint4& v, float (&x)[N]) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = clean(f.x), x[2 * i + 1] = clean(f.y);
    }
  }
  static __device__ __forceinline__ float one(const __half* p) { return clean(__half2float(*p)); }
};

__device__ __forceinline__ double max_double(double a, double b) { return a > b ? a : b; }

__device__ __forceinline__ unsigned long long ld_cluster_u64(uint32_t addr) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

// The order of doubles as unsigned integers, and back.
__device__ __forceinline__ Key ordered(double x) {
  const Key u = Key(__double_as_longlong(x == 0.0 ? 0.0 : x));
  return (u >> 63) ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double unordered(Key o) { return __longlong_as_double((o >> 63) ? (long long)(o & ~(1ull << 63)) : (long long)~o); }

template <typename T>
__global__ void __launch_bounds__(THREADS, 4)
kf_beam_select(const T* __restrict__ logits, long long stride_b, long long stride_w, const float* __restrict__ scores,
               const uint8_t* __restrict__ finished, int W, int V, long long eos, long long pad, float* __restrict__ out_scores,
               long long* __restrict__ out_parents, long long* __restrict__ out_tokens, uint8_t* __restrict__ out_finished) {
  constexpr int N = Logits<T>::N;
  constexpr float LOG2E = 1.4426950408889634f;
  constexpr int UNROLL = 8;
  struct Part {
    double m, sum;
    Key keys[MAX_BEAMS];
  };
  __shared__ Part parts[MAX_PARTS];
  __shared__ uint32_t tops[WARPS][MAX_BEAMS];      // each warp's threads by their largest logit
  __shared__ double ms[WARPS], sums[WARPS];
  __shared__ uint32_t bound;
  __shared__ int n_readers, n_found;
  __shared__ uint16_t readers[THREADS];
  __shared__ Key found[WARPS * MAX_BEAMS];         // ROOM candidates, or the warps' lists
  __shared__ double total[MAX_BEAMS * MAX_BEAMS];  // [W][W], best first, -inf: none
  __shared__ uint32_t token[MAX_BEAMS * MAX_BEAMS];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int ctas = int(cluster_nctaid()), rank = int(cluster_ctarank());
  const long long b = blockIdx.x / ctas, first = b * W;
  // Beams whose logits count.  One without a score above -inf (or with NaN) has no candidates, a finished one has itself.
  const bool alive = lane < W && scores[first + lane] > -INFINITY;
  const bool done = lane < W && finished != nullptr && finished[first + lane];
  const uint32_t live = __ballot_sync(0xffffffffu, alive && !done);
  const int per = V / N + 1;                       // vectors of a row, at most
  const long long all = (long long)__popc(live) * per;
  const int working = all < ctas ? int(all) : ctas;   // CTAs that have a range, and one that is not empty
  const long long r0 = rank < working ? all * rank / working : 0, r1 = rank < working ? all * (rank + 1) / working : 0;

  int part = 0;
  for (long long pos = r0; pos < r1; ++part) {
    const int nth = int(pos / per), v0 = int(pos % per);
    const int v_end = int(r1 - pos < per - v0 ? v0 + (r1 - pos) : per);
    pos += v_end - v0;
    const int w = __fns(live, 0, nth + 1);
    const T* x0 = logits + b * stride_b + w * stride_w;
    // vectors from the row's first 16-byte boundary on; what is left at both ends goes with the first vector, a value a thread
    const int misaligned = int(reinterpret_cast<uintptr_t>(x0) & 15) / int(sizeof(T));
    const int head = misaligned ? min(V, N - misaligned) : 0;
    const int vectors = (V - head) / N, tail0 = head + vectors * N;
    const int v1 = min(v_end, vectors);
    const uint4* vec = reinterpret_cast<const uint4*>(x0 + head);
    auto single = [&](int t) { return v0 != 0 ? -1 : t < head ? t : t >= N && t - N < V - tail0 ? tail0 + t - N : -1; };

    float m = -INFINITY, sum = 0.f;
    if (tid < 2 * N) {
      const int i = single(tid);
      const float x = i >= 0 ? Logits<T>::one(x0 + i) : -INFINITY;
      if (x > -INFINITY) m = x, sum = 1.f;
    }
    for (int base = v0 + tid; base < v1; base += THREADS * UNROLL) {
      uint4 raw[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
        if (base + u * THREADS < v1) raw[u] = vec[base + u * THREADS];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        if (base + u * THREADS >= v1) break;
        float x[N];
        Logits<T>::load(raw[u], x);
        float mx = x[0];
#pragma unroll
        for (int j = 1; j < N; ++j) mx = max_of(mx, x[j]);
        if (mx > m) {
          sum = m == -INFINITY ? 0.f : sum * exp2_fast((m - mx) * LOG2E);
          m = mx;
        } else {
          m = max_of(m, mx);   // apart where both are below the smallest normal number, which the compare takes for zeros
        }
        const float from = m == -INFINITY ? 0.f : m;
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < N; ++j) s[j & 1] += exp2_fast((x[j] - from) * LOG2E);
        sum += s[0] + s[1];
      }
    }

    // ---- the sum, and each warp's threads in order
    double wm = double(m), ws = double(sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) wm = max_double(wm, __shfl_xor_sync(0xffffffffu, wm, o));
    if (m > -INFINITY) ws *= double(exp2_fast(float(double(m) - wm) * LOG2E));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
    if (lane == 0) ms[warp] = wm, sums[warp] = ws;
    const uint32_t best = m > -INFINITY ? ordered(m) : 0u;   // 0: none
    const uint32_t in_order = sorted(best);
    tops[warp][lane] = in_order;
    if (tid == 0) n_readers = n_found = 0;
    __syncthreads();
    // ---- the W-th largest of the threads' largest: that with W - 1 before it (equal ones in the order of the warps)
    if (lane < W) {
      int before = lane;
      for (int x = 0; x < WARPS; ++x) {
        if (x == warp) continue;
        // the lists are sorted: how many of the first W come before mine
        for (int i = 0; i < W; ++i) {
          const uint32_t other = tops[x][i];
          if (other < in_order || (other == in_order && x > warp)) break;
          ++before;
        }
      }
      if (before == W - 1) bound = in_order;
    }
    __syncthreads();
    if (best != 0u && best >= bound) readers[atomicAdd(&n_readers, 1)] = uint16_t(tid);
    __syncthreads();
    // ---- the logits of these threads again
    const int n = n_readers;
    const uint32_t least = bound;
    for (int i = warp; i < n; i += WARPS) {
      const int t = readers[i];
      for (int base = v0 + t; base < v1; base += THREADS * 32) {
        const int at = base + lane * THREADS;
        if (at < v1) {
          float x[N];
          Logits<T>::load(vec[at], x);
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (x[j] > -INFINITY && ordered(x[j]) >= least) {
              const int to = atomicAdd(&n_found, 1);
              if (to < ROOM) found[to] = make_key(x[j], uint32_t(head + at * N + j));
            }
        }
      }
      if (lane == 0 && t < 2 * N && single(t) >= 0) {
        const float x = Logits<T>::one(x0 + single(t));
        if (x > -INFINITY && ordered(x) >= least) {
          const int to = atomicAdd(&n_found, 1);
          if (to < ROOM) found[to] = make_key(x, uint32_t(single(t)));
        }
      }
    }
    __syncthreads();
    const int candidates = n_found;
    Key mine = 0;
    if (candidates <= ROOM) {
      if (warp == 0)
        for (int i = 0; i < candidates; i += 32) {
          const Key k = sorted(i + lane < candidates ? found[i + lane] : 0);
          mine = i ? merged(mine, k) : k;
        }
    } else {
      // so many equal logits that there is no room: every warp through the whole of its vectors
      TopList top;
      for (int base = v0 + warp * 32; base < v1; base += THREADS) {
        const int at = base + lane;
        float x[N];
        if (at < v1) Logits<T>::load(vec[at], x);
#pragma unroll
        for (int j = 0; j < N; ++j)
          top.offer(at < v1 && x[j] > -INFINITY && ordered(x[j]) >= least ? make_key(x[j], uint32_t(head + at * N + j)) : 0, W);
      }
      if (warp == 0) {
        const int i = lane < 2 * N ? single(lane) : -1;
        const float x = i >= 0 ? Logits<T>::one(x0 + i) : -INFINITY;
        top.offer(x > -INFINITY ? make_key(x, uint32_t(i)) : 0, W);
      }
      found[warp * MAX_BEAMS + lane] = top.mine;
      __syncthreads();
      if (warp == 0)
        for (int i = 0; i < WARPS; ++i) mine = i ? merged(mine, found[i * MAX_BEAMS + lane]) : found[lane];
    }
    if (warp == 0) {
      parts[part].keys[lane] = mine;
      double pm = lane < WARPS ? ms[lane] : -INFINITY;
      const double own = pm;
#pragma unroll
      for (int o = WARPS / 2; o > 0; o >>= 1) pm = max_double(pm, __shfl_xor_sync(0xffffffffu, pm, o));
      double ps = lane < WARPS && own > -INFINITY ? sums[lane] * exp2((own - pm) * LOG2E_D) : 0.0;
#pragma unroll
      for (int o = WARPS / 2; o > 0; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
      if (lane == 0) parts[part].m = pm, parts[part].sum = ps;
    }
    __syncthreads();
  }

  cluster_sync_all();
  // ---- the first CTA joins what the cluster found, a warp a beam
  const double NONE = -INFINITY;
  if (rank == 0) {
    for (int w = warp; w < W; w += WARPS) {
      const bool w_alive = scores[first + w] > -INFINITY;
      if ((live >> w) & 1u) {
        const int nth = __popc(live & ((1u << w) - 1u));
        const long long u0 = (long long)nth * per, u1 = u0 + per - 1;
        const int c0 = int(((u0 + 1) * working - 1) / all), c1 = int(((u1 + 1) * working - 1) / all);   // CTAs that hold its first and last vector
        auto part_of = [&](int c) {
          const long long begin = all * c / working;
          return mapa_shared(smem_u32(&parts[nth - int(begin / per)]), uint32_t(c));
        };
        double m = NONE, sum = 0.0, own_m = NONE, own_sum = 0.0;
        if (lane <= c1 - c0) {
          const uint32_t at = part_of(c0 + lane);
          own_m = __longlong_as_double((long long)ld_cluster_u64(at));
          own_sum = __longlong_as_double((long long)ld_cluster_u64(at + 8));
        }
        m = own_m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max_double(m, __shfl_xor_sync(0xffffffffu, m, o));
        sum = own_m > NONE ? own_sum * exp2((own_m - m) * LOG2E_D) : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const double lse = m + log(sum);
        Key mine = 0;
        const int count = (c1 - c0 + 1) * W;
        for (int i = 0; i < count; i += 32) {
          Key k = 0;
          if (i + lane < count) k = ld_cluster_u64(part_of(c0 + (i + lane) / W) + 16 + 8 * ((i + lane) % W));
          k = sorted(k);
          mine = i ? merged(mine, k) : k;
        }
        if (lane < W) {
          total[w * W + lane] = mine ? double(scores[first + w]) + (double(key_value(mine)) - lse) : NONE;
          token[w * W + lane] = key_index(mine);
        }
      } else if (lane < W) {
        total[w * W + lane] = lane == 0 && w_alive ? double(scores[first + w]) : NONE;   // finished, or nothing
      }
    }
  }
  __syncthreads();
  if (rank == 0 && warp == 0) {
    // lane = beam; its best candidate that is not taken yet.  The score in two halves: the larger, of equal ones the lower beam.
    int at = 0, parent = lane, place = -1;
    const Key none = ordered(NONE);
    Key mine = lane < W ? ordered(total[lane * W]) : none, score = none;
    for (int r = 0; r < W; ++r) {
      const uint32_t hi = __reduce_max_sync(0xffffffffu, uint32_t(mine >> 32));
      const uint32_t lo = __reduce_max_sync(0xffffffffu, uint32_t(mine >> 32) == hi ? uint32_t(mine) : 0u);
      const Key best = (Key(hi) << 32) | lo;
      if (best <= none) break;
      const int who = __ffs(__ballot_sync(0xffffffffu, mine == best)) - 1;
      const int taken = __shfl_sync(0xffffffffu, at, who);
      if (lane == r) score = best, parent = who, place = taken;
      if (lane == who) {
        ++at;
        mine = at < W ? ordered(total[lane * W + at]) : none;
      }
    }
    const uint32_t ends = __ballot_sync(0xffffffffu, done);
    if (lane < W) {
      const bool ended = place >= 0 && ((ends >> parent) & 1u);
      const long long t = place < 0 || ended ? pad : (long long)token[parent * W + place];
      out_scores[first + lane] = float(unordered(score));
      out_parents[first + lane] = parent;
      out_tokens[first + lane] = t;
      out_finished[first + lane] = ended || (place >= 0 && t == eos);
    }
  }
  cluster_sync_all();   // no CTA leaves while the first reads its shared memory
}

template <typename T>
static int launch_select(const void* logits, long long stride_b, long long stride_w, const float* scores, const uint8_t* finished, int B, int W, int V,
                         long long eos, long long pad, float* out_scores, long long* out_parents, long long* out_tokens, uint8_t* out_finished,
                         int num_sms, cudaStream_t stream) {
  auto kern = kf_beam_select<T>;
  cudaLaunchConfig_t cfg = {};
  const int ctas = MIN_CTAS;
  if ((long long)B * ctas > 0x7fffffffLL) return 6;
  cfg.gridDim = dim3((unsigned)(B * ctas));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, (const T*)logits, stride_b, stride_w, scores, finished, W, V, eos, pad, out_scores, out_parents,
                                     out_tokens, out_finished);
  return e == cudaSuccess ? 0 : 500 + (int)e;
}

// ------------------------------------------------------------------ reorder
struct State {
  const uint8_t* src;
  uint8_t* dst;
  long long src_b, src_w, dst_b, dst_w;   // bytes
  long long bytes;                        // of a beam that follow it
};
constexpr int MAX_STATES = 56;            // with the rest of the arguments below 4 KB
struct States {
  State s[MAX_STATES];
  long long first[MAX_STATES + 1];        // prefix sums of columns x prompts
};

// T: the widest word that all addresses and steps are multiples of.  A column is one word; the last column of a state may hold fewer
// bytes than a word and is moved byte by byte.
template <typename T, int W>
__global__ void __launch_bounds__(256)
kf_beam_reorder(const __grid_constant__ States st, int n, int beams, const void* __restrict__ parents, int wide) {
  const long long total = st.first[n];
  int s = 0;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
    while (i >= st.first[s + 1]) ++s;
    const State& a = st.s[s];
    const long long columns = (a.bytes + sizeof(T) - 1) / (long long)sizeof(T);
    const long long b = (i - st.first[s]) / columns, off = (i - st.first[s]) % columns * (long long)sizeof(T);
    const uint8_t* src = a.src + b * a.src_b + off;
    uint8_t* dst = a.dst + b * a.dst_b + off;
    const bool in_place = a.src == a.dst;
    const int left = int(a.bytes - off < (long long)sizeof(T) ? a.bytes - off : (long long)sizeof(T));
    T v[W];
    bool move[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      move[w] = false;
      if (w < beams) {
        const long long p = wide ? reinterpret_cast<const long long*>(parents)[b * beams + w]
                                 : (long long)reinterpret_cast<const int*>(parents)[b * beams + w];
        // a parent that is no beam: the state stays as it is
        move[w] = p >= 0 && p < beams && !(in_place && p == w);
        if (move[w]) {
          const uint8_t* from = src + p * a.src_w;
          if (left == (int)sizeof(T)) {
            v[w] = *reinterpret_cast<const T*>(from);
          } else {
            uint8_t* bytes = reinterpret_cast<uint8_t*>(&v[w]);
            for (int j = 0; j < (int)sizeof(T); ++j)
              if (j < left) bytes[j] = from[j];
          }
        }
      }
    }
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (move[w]) {
        uint8_t* to = dst + w * a.dst_w;
        if (left == (int)sizeof(T)) {
          *reinterpret_cast<T*>(to) = v[w];
        } else {
          const uint8_t* bytes = reinterpret_cast<const uint8_t*>(&v[w]);
          for (int j = 0; j < (int)sizeof(T); ++j)
            if (j < left) to[j] = bytes[j];
        }
      }
  }
}

template <typename T>
static void launch_reorder(const States& st, int n, int beams, const void* parents, int wide, int num_sms, cudaStream_t stream) {
  const long long need = (st.first[n] + 255) / 256;
  const unsigned grid = (unsigned)(need < 8LL * num_sms ? need : 8LL * num_sms);
  if (beams <= 4) kf_beam_reorder<T, 4><<<grid, 256, 0, stream>>>(st, n, beams, parents, wide);
  else if (beams <= 8) kf_beam_reorder<T, 8><<<grid, 256, 0, stream>>>(st, n, beams, parents, wide);
  else if (beams <= 16) kf_beam_reorder<T, 16><<<grid, 256, 0, stream>>>(st, n, beams, parents, wide);
  else kf_beam_reorder<T, 32><<<grid, 256, 0, stream>>>(st, n, beams, parents, wide);
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
  if (B < 1 || W < 1 || W > MAX_BEAMS || V < 1) return 3;
  auto go = [&](auto launch) {
    return launch(logits, stride_b, stride_w, (const float*)scores, (const uint8_t*)finished, B, W, V, eos, pad, (float*)out_scores,
                  (long long*)out_parents, (long long*)out_tokens, (uint8_t*)out_finished, num_sms, (cudaStream_t)stream);
  };
  if (type == 0) return go(launch_select<__nv_bfloat16>);
  if (type == 1) return go(launch_select<float>);
  if (type == 2) return go(launch_select<__half>);
  return 4;
}

int kf_beam_max_states() { return kf::beam::MAX_STATES; }

// table: 7 numbers a state (src, dst, and in bytes: steps of src and dst from prompt to prompt and beam to beam as src_b, src_w, dst_b,
// dst_w, and the length that moves).  parents (B, beams), int64 or (wide == 0) int32.  dst is src itself or does not overlap it.
int kf_beam_reorder(const long long* table, int n, int B, int beams, const void* parents, int wide, int num_sms, void* stream) {
  using namespace kf::beam;
  if (n < 1 || n > MAX_STATES || B < 1 || beams < 1 || beams > MAX_BEAMS) return 3;
  States st;
  unsigned long long all = 0;
  for (int i = 0; i < n; ++i) {
    const long long* t = table + 7 * i;
    st.s[i] = State{(const uint8_t*)t[0], (uint8_t*)t[1], t[2], t[3], t[4], t[5], t[6]};
    if (t[6] < 0) return 3;
    for (int j = 0; j < 6; ++j) all |= (unsigned long long)t[j];
  }
  const int word = !(all & 15) ? 16 : !(all & 7) ? 8 : !(all & 3) ? 4 : !(all & 1) ? 2 : 1;
  st.first[0] = 0;
  for (int i = 0; i < n; ++i) st.first[i + 1] = st.first[i] + (st.s[i].bytes + word - 1) / word * B;
  if (st.first[n] == 0) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (word == 16) launch_reorder<uint4>(st, n, beams, parents, wide, num_sms, s);
  else if (word == 8) launch_reorder<unsigned long long>(st, n, beams, parents, wide, num_sms, s);
  else if (word == 4) launch_reorder<uint32_t>(st, n, beams, parents, wide, num_sms, s);
  else if (word == 2) launch_reorder<uint16_t>(st, n, beams, parents, wide, num_sms, s);
  else launch_reorder<uint8_t>(st, n, beams, parents, wide, num_sms, s);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 400 + (int)e;
}

}  // extern "C"
