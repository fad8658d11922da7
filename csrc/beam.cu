// Beam search: the best W continuations of W beams, and the states that follow them.
//
// kf_beam_select.  Of each prompt's W beams with scores s_w and logits l_w (V values each) the W best pairs (w, t) by
//     s_w + l_w[t] - log sum_t' exp(l_w[t']) .
// Within a beam the order of candidates is that of its logits, so W tokens of each beam are all that can be among the best, and one pass
// over the logits finds them together with the sum: kf_beam_rows.  Every warp keeps the W largest logits that it has met, one per lane,
// as 64-bit keys (the logit's bits in an order-preserving form, then the complement of its index: of equal logits the lowest index is
// the largest key).  A vector of logits costs a packed maximum and a compare with the warp's W-th largest; only what is above it is
// inserted, W ln(n / W) times for n values in random order.  The sum runs over exp(x - m) with m the largest so far, in fp32 per thread
// (at most a few hundred terms each) and in 64 bits from there on, because candidates of different beams may lie close together.  The
// difference is taken before the factor log2 e: rows of the type's lowest value have exponents of zero like any others, and no product
// overflows.
// What bounds it: the logits are read once.  A row is split over blocks so that a few rows fill the GPU too; kf_beam_merge, one block a
// prompt, joins the splits, one warp a beam, and picks W times the best of the beams' heads.
//
// kf_beam_reorder.  state[b, w] = state[b, parent[b, w]] for all states in one launch.  A thread owns 16 bytes of a column: it reads
// the column's W values and then writes them, so that parents may be any selection of beams, also in place, without a second buffer.
#include "common.cuh"
#include "skinny_common.cuh"

#include <cuda_fp16.h>

namespace kf {
namespace beam {

constexpr int MAX_BEAMS = 32;   // a warp's list is one key per lane
constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;
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

// The largest `width` keys that a warp has met, lane i the i-th (0 = none).
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

// What a block leaves of its part of a row: the largest logit m and the sum of exp(x - m) over the part; its keys lie beside.
struct Part {
  double sum, m;
};
// Of the kernel before this one (see ld_after_wait).
__device__ __forceinline__ Part load_part(const Part* p) {
  Part v;
  asm volatile("ld.global.v2.f64 {%0, %1}, [%2];" : "=d"(v.sum), "=d"(v.m) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ Key load_key(const Key* p) {
  Key v;
  asm volatile("ld.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
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

// A beam that has candidates: a score above -inf (not NaN).  A finished one has a single candidate and needs no pass over its logits.
__device__ __forceinline__ bool alive(const float* scores, long long row) { return scores[row] > -INFINITY; }

template <typename T>
__global__ void __launch_bounds__(THREADS)
kf_beam_rows(const T* __restrict__ logits, long long stride_b, long long stride_w, const float* __restrict__ scores,
             const uint8_t* __restrict__ finished, int W, int V, int splits, int chunk, Part* __restrict__ parts, Key* __restrict__ keys) {
  constexpr int N = Logits<T>::N;
  constexpr float LOG2E = 1.4426950408889634f;
  __shared__ Key lists[WARPS][MAX_BEAMS];
  __shared__ float ms[WARPS];
  __shared__ double sums[WARPS];
  grid_dep_launch();
  const long long row = blockIdx.x / splits;
  const int split = int(blockIdx.x % splits);
  if (!alive(scores, row) || (finished && finished[row])) return;   // kf_beam_merge asks nothing of this row's parts
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* x0 = logits + (row / W) * stride_b + (row % W) * stride_w;

  TopList top;
  float m = -INFINITY, sum = 0.f;
  auto add = [&](float x) {   // one value (lanes without one pass -inf)
    const float mn = fmaxf(m, x);
    if (mn == -INFINITY) return;
    sum = (m == -INFINITY ? 0.f : sum * exp2_fast((m - mn) * LOG2E)) + exp2_fast((x - mn) * LOG2E);
    m = mn;
  };
  // the row from its first 16-byte boundary on in vectors; what is left at both ends is the first split's
  const int head = min(V, int((16 - (reinterpret_cast<uintptr_t>(x0) & 15)) & 15) / int(sizeof(T)));
  const int vectors = (V - head) / N;
  const int tail0 = head + vectors * N;
  if (split == 0 && warp == 0) {
    int i = -1;
    if (lane < head) i = lane;
    else if (lane >= 16 && tail0 + lane - 16 < V) i = tail0 + lane - 16;
    const float x = i >= 0 ? Logits<T>::one(x0 + i) : -INFINITY;
    add(x);
    top.offer(x > -INFINITY ? make_key(x, uint32_t(i)) : 0, W);
  }
  const uint4* vec = reinterpret_cast<const uint4*>(x0 + head);
  const int v0 = split * chunk, v1 = min(vectors, v0 + chunk);
  constexpr int UNROLL = 4;
  for (int base = v0 + warp * 32; base < v1; base += THREADS * UNROLL) {
    uint4 raw[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int i = base + u * THREADS + lane;
      if (i < v1) raw[u] = __ldcs(vec + i);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int i = base + u * THREADS + lane;
      float x[N];
      if (i < v1) {
        Logits<T>::load(raw[u], x);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = -INFINITY;
      }
      float mx = x[0];
#pragma unroll
      for (int j = 1; j < N; ++j) mx = max_of(mx, x[j]);
      if (mx > m) {
        sum *= m == -INFINITY ? 0.f : exp2_fast((m - mx) * LOG2E);
        m = mx;
      }
      const float b = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int j = 0; j < N; ++j) sum += exp2_fast((x[j] - b) * LOG2E);
      if (__any_sync(0xffffffffu, mx > -INFINITY && ordered(mx) >= uint32_t(top.worst >> 32))) {
#pragma unroll
        for (int j = 0; j < N; ++j) top.offer(x[j] > -INFINITY ? make_key(x[j], uint32_t(head + i * N + j)) : 0, W);
      }
    }
  }

  // the warp's sum, then the block's
  float wm = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
  double ws = m == -INFINITY ? 0.0 : double(sum) * exp2((double(m) - double(wm)) * LOG2E_D);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
  if (lane == 0) ms[warp] = wm, sums[warp] = ws;
  lists[warp][lane] = top.mine;
  __syncthreads();
  if (warp != 0) return;
  for (int i = 1; i < WARPS; ++i) top.offer(lists[i][lane], W);
  if (lane < W) keys[(long long)blockIdx.x * W + lane] = top.mine;
  if (lane == 0) {
    float bm = -INFINITY;
    for (int i = 0; i < WARPS; ++i) bm = fmaxf(bm, ms[i]);
    double bs = 0.0;
    for (int i = 0; i < WARPS; ++i)
      if (ms[i] > -INFINITY) bs += sums[i] * exp2((double(ms[i]) - double(bm)) * LOG2E_D);
    parts[blockIdx.x] = Part{bs, double(bm)};
  }
}

// One block a prompt, one warp a beam.
__global__ void kf_beam_merge(const Part* parts, const Key* keys, const float* __restrict__ scores,
                              const uint8_t* __restrict__ finished, int W, int splits, long long eos, long long pad,
                              float* __restrict__ out_scores, long long* __restrict__ out_parents, long long* __restrict__ out_tokens,
                              uint8_t* __restrict__ out_finished) {
  extern __shared__ __align__(8) uint8_t smem[];
  double* total = reinterpret_cast<double*>(smem);                        // [W][W], best first, -inf: none
  uint32_t* token = reinterpret_cast<uint32_t*>(total + W * W);           // [W][W]
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * W + w;
  grid_dep_wait();
  const double NONE = -INFINITY;
  const bool done = finished && finished[row];
  if (alive(scores, row) && !done) {
    const Part* p = parts + row * splits;
    const Key* k = keys + row * splits * W;
    double m = -INFINITY;
    for (int i = lane; i < splits; i += 32) m = fmax(m, load_part(p + i).m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
    double sum = 0.0;
    for (int i = lane; i < splits; i += 32) {
      const Part x = load_part(p + i);
      if (x.m > -INFINITY) sum += x.sum * exp2((x.m - m) * LOG2E_D);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const double lse = m + log(sum);
    TopList top;
    for (int i = 0; i < splits * W; i += 32) top.offer(i + lane < splits * W ? load_key(k + i + lane) : 0, W);
    if (lane < W) {
      total[w * W + lane] = top.mine ? double(scores[row]) + (double(key_value(top.mine)) - lse) : NONE;
      token[w * W + lane] = key_index(top.mine);
    }
  } else if (lane < W) {
    total[w * W + lane] = done && lane == 0 && alive(scores, row) ? double(scores[row]) : NONE;
  }
  __syncthreads();
  if (w != 0) return;
  // lane = beam; its best candidate that is not taken yet
  int at = 0, parent = lane, place = -1;
  double mine = lane < W ? total[lane * W] : NONE, score = NONE;
  for (int r = 0; r < W; ++r) {
    double best = mine;
    int who = lane;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double other = __shfl_xor_sync(0xffffffffu, best, o);
      const int whose = __shfl_xor_sync(0xffffffffu, who, o);
      if (other > best || (other == best && whose < who)) best = other, who = whose;
    }
    if (best == NONE) break;
    const int taken = __shfl_sync(0xffffffffu, at, who);
    if (lane == r) score = best, parent = who, place = taken;
    if (lane == who) {
      ++at;
      mine = at < W ? total[lane * W + at] : NONE;
    }
  }
  if (lane >= W) return;
  const long long first = (long long)blockIdx.x * W, to = first + lane;
  const bool ended = place >= 0 && finished && finished[first + parent];
  const long long t = place < 0 || ended ? pad : (long long)token[parent * W + place];
  out_scores[to] = float(score);
  out_parents[to] = parent;
  out_tokens[to] = t;
  out_finished[to] = ended || (place >= 0 && t == eos);
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

// How many blocks share a row of V logits.
int kf_beam_splits(long long rows, int V, int size, int num_sms) {
  // eight blocks an SM at most; a block has at least one vector of 16 bytes for each of its threads
  const long long most = ((long long)V * size + 16 * kf::beam::THREADS - 1) / (16 * kf::beam::THREADS);
  long long s = (8LL * num_sms) / (rows > 0 ? rows : 1);
  if (s > most) s = most;
  return s < 1 ? 1 : (int)s;
}

// logits (B, W, V) with strides in elements and V side by side; type 0 bf16, 1 fp32, 2 fp16.  scores (B, W) fp32, finished (B, W) bytes
// or null.  parts: splits * B * W * (16 + 8 W) bytes of scratch, on 16.  Writes scores, parents, tokens and finished (B, W).
int kf_beam_select(const void* logits, int type, long long stride_b, long long stride_w, const void* scores, const void* finished, int B, int W,
                   int V, long long eos, long long pad, void* parts, int splits, void* out_scores, void* out_parents, void* out_tokens,
                   void* out_finished, void* stream) {
  using namespace kf::beam;
  const long long rows = (long long)B * W;
  if (B < 1 || W < 1 || W > MAX_BEAMS || V < 1 || splits < 1 || rows * splits > 0x7fffffffLL) return 3;
  cudaStream_t st = (cudaStream_t)stream;
  const int size = type == 1 ? 4 : 2, per = 16 / size;
  const int vectors = V / per + 1;
  const int chunk = (vectors + splits - 1) / splits;
  Part* p = (Part*)parts;
  Key* k = (Key*)(p + rows * splits);
  const unsigned grid = (unsigned)(rows * splits);
  const float* sc = (const float*)scores;
  const uint8_t* fin = (const uint8_t*)finished;
  if (type == 0)
    kf_beam_rows<__nv_bfloat16><<<grid, THREADS, 0, st>>>((const __nv_bfloat16*)logits, stride_b, stride_w, sc, fin, W, V, splits, chunk, p, k);
  else if (type == 1)
    kf_beam_rows<float><<<grid, THREADS, 0, st>>>((const float*)logits, stride_b, stride_w, sc, fin, W, V, splits, chunk, p, k);
  else if (type == 2)
    kf_beam_rows<__half><<<grid, THREADS, 0, st>>>((const __half*)logits, stride_b, stride_w, sc, fin, W, V, splits, chunk, p, k);
  else
    return 4;
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return 400 + (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)B);
  cfg.blockDim = dim3((unsigned)W * 32);
  cfg.dynamicSmemBytes = size_t(W) * W * 12;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kf_beam_merge, (const Part*)p, (const Key*)k, sc, fin, W, splits, eos, pad, (float*)out_scores,
                         (long long*)out_parents, (long long*)out_tokens, (uint8_t*)out_finished);
  return e == cudaSuccess ? 0 : 500 + (int)e;
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
