// What a row of logits says about tokens: the log probability of a given one, its rank, the row's entropy, and the most likely
// alternatives with their log probabilities.
//
//   lse = log sum_j exp(x_j),   log p_t = x_t - lse,   H = -sum_j p_j log p_j = log s - (sum_j d_j exp(d_j)) / s
//   with d_j = x_j - max, s = sum_j exp(d_j);   rank of t = how many columns come before it (larger, or equal with a lower id).
//
// Both terms of H are >= 0, so nothing cancels.  A row whose every column is -inf has no distribution: its log probabilities
// are -inf and its entropy 0.  A row that holds NaN or +inf gives NaN; a token whose own logit is NaN has no rank (-1).  NaN comes
// behind -inf among the alternatives.
//
// Shape.  A row is read once.  A block walks its slice of the row in chunks of 8,192 columns, 32 in the registers of each
// thread (the next chunk's on their way), and keeps per thread the running maximum m, s and u = sum d exp(d) (a new maximum moves
// both: u' = f (u + (m - m') s), s' = f s, f = exp(m - m')).  A cluster of up to 16 blocks shares a row when there are few
// rows; each leaves its numbers in the first block's shared memory, so nothing passes through a workspace and one launch does it all.
// Alternatives: the block keeps a list of keys that can still be among its k best, in shared memory, and a value tau that a
// column must exceed to join them.  The first chunk is cut by a bound that at least k of its columns reach (`warp_bound`) and
// leaves the exact k-th value as tau.  From then on a column costs one comparison (of the thread's maximum), and a random row
// brings k * 8,192 / (columns seen) keys a chunk; a list grown long is pruned to its k best, which raises tau.
// What bounds it: memory for long 32-bit rows without alternatives (512 x 256,000 in 89 to 92 us, 5.7 to 5.9 TB/s; bfloat16 78 us, the arithmetic
// of a column); with them the first chunk's bound and ranking and the row's last ranking, which its loads do not cover (L2 flushed before:
// 512 rows with 20 alternatives 131 us, 64 rows 31 to 33, one row 14 to 16).
#include "row_stats.cuh"

namespace {

using namespace kf_row;

constexpr int TOP_MAX = 64;
constexpr int NT = 256, WARPS = NT / 32;
constexpr int PER_THREAD = 32;                               // columns of a chunk in a thread's registers
constexpr int CHUNK = NT * PER_THREAD;
constexpr int MAX_SLICES = 16;
constexpr int KEY_CAP = NT * 8 + TOP_MAX;                    // keys held at most: a vector of every thread beside the k best
constexpr int TAIL_MAX = 7;                                  // columns behind a row's last vector; the list has room for them besides
constexpr int FEW_KEYS = 256;                                // up to here keys are ranked by counting the larger ones at once

__device__ __forceinline__ unsigned orderable(float v) {     // larger float <=> larger unsigned; -0 as +0; NaN below everything
  const unsigned b = __float_as_uint(v == 0.f ? 0.f : v);
  return v != v ? 0u : ((b & 0x80000000u) ? ~b : (b | 0x80000000u));
}
// (value, id) as one number: a larger key comes first, no two are equal, zero is none of them
__device__ __forceinline__ u64 rank_key(float v, unsigned id) { return ((u64)orderable(v) << 32) | (u64)(0xFFFFFFFFu - id); }
__device__ __forceinline__ float rank_value(u64 key) {
  const unsigned o = (unsigned)(key >> 32);
  return o == 0u ? __int_as_float(0x7fffffff) : __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ int rank_id(u64 key) { return (int)(0xFFFFFFFFu - (unsigned)key); }

// Sixteen bytes of a row as floats
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  static constexpr unsigned MASKED = 0xff800000u;
  static __device__ __forceinline__ float get(const uint4& v, int i) {
    return __uint_as_float(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
  }
  static __device__ __forceinline__ float half_of(unsigned word, int) { return __uint_as_float(word); }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr unsigned MASKED = 0xff80ff80u;
  static __device__ __forceinline__ float get(const uint4& v, int i) {
    const unsigned w = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
    return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ float half_of(unsigned word, int i) { return __uint_as_float((i & 1) ? (word & 0xffff0000u) : (word << 16)); }
};
// Column `at` (0..31) of those a thread holds: a tree of selections, since registers have no addresses
template <typename T, int NV>
__device__ __forceinline__ float pick(const uint4 (&raw)[NV], int at) {
  constexpr int PER_WORD = 4 / sizeof(T);
  unsigned w[NV * 4];
#pragma unroll
  for (int j = 0; j < NV; ++j) { w[4 * j] = raw[j].x; w[4 * j + 1] = raw[j].y; w[4 * j + 2] = raw[j].z; w[4 * j + 3] = raw[j].w; }
  int word = at / PER_WORD;
#pragma unroll
  for (int n = NV * 4; n > 1; n /= 2) {
#pragma unroll
    for (int i = 0; i < n / 2; ++i) w[i] = (word & 1) ? w[2 * i + 1] : w[2 * i];
    word >>= 1;
  }
  return Vec<T>::half_of(w[0], at);
}

struct Shared {
  Stats stats[WARPS];
  int before[WARPS];
  float bound[WARPS];
  int n_keys;
  u64 sorted[TOP_MAX];
  u64 keys[KEY_CAP + TAIL_MAX];
};
struct ClusterShared {                                        // what the row's blocks leave with the first one
  Stats stats[MAX_SLICES];
  int before[MAX_SLICES];
  u64 keys[MAX_SLICES * TOP_MAX];
};

// A value that at least k of the block's threads' numbers reach (-inf: there may be fewer): with q = ceil(k / warps), the smallest
// of the warps' q-th largest.  A number's rank in its warp is how many lanes hold a larger one, lower lanes first among equals.
// All threads call it.
__device__ __noinline__ float warp_bound(float mine, int k, Shared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int q = (k + WARPS - 1) / WARPS;
  int rank = 0;
#pragma unroll
  for (int o = 1; o < 32; ++o) {
    const float other = __shfl_sync(0xffffffffu, mine, (lane + o) & 31);
    rank += (other > mine || (other == mine && ((lane + o) & 31) < lane)) ? 1 : 0;
  }
  if (rank == q - 1) sh.bound[warp] = mine;
  __syncthreads();
  float b = sh.bound[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) b = fminf(b, sh.bound[w]);
  __syncthreads();
  return b;
}

// Of the keys in the list [0, n), those of at least `bound` and whose ids are not in [id0, id1), moved to its front; returns how
// many.  All threads call it.
__device__ __noinline__ int compact(int n, float bound, unsigned id0, unsigned id1, Shared& sh) {
  constexpr int MINE = (KEY_CAP + TAIL_MAX + NT - 1) / NT;
  const int tid = threadIdx.x;
  u64 mine[MINE];
#pragma unroll
  for (int j = 0; j < MINE; ++j) mine[j] = tid + j * NT < n ? sh.keys[tid + j * NT] : 0ull;
  __syncthreads();
  if (tid == 0) sh.n_keys = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < MINE; ++j) {
    const unsigned id = (unsigned)rank_id(mine[j]);
    if (mine[j] != 0ull && rank_value(mine[j]) >= bound && (id < id0 || id >= id1)) sh.keys[atomicAdd(&sh.n_keys, 1)] = mine[j];
  }
  __syncthreads();
  const int left = sh.n_keys;
  __syncthreads();
  return left;
}

// The k best of keys[0, n) to sh.sorted, in order: a key's place is how many are larger; `share` neighbouring lanes count for
// one key.  Zeros are absent ones.  All threads call it.
__device__ __forceinline__ void rank_keys(const u64* keys, int n, int k, Shared& sh) {
  int share = 1;
  while (share < 8 && n * share * 2 <= NT) share *= 2;
  for (int i0 = 0; i0 * share < n * share; i0 += NT / share) {
    const int i = i0 + threadIdx.x / share;
    const u64 key = i < n ? keys[i] : 0ull;
    int rank = 0;
#pragma unroll 4
    for (int j = threadIdx.x % share; j < n; j += share) rank += keys[j] > key ? 1 : 0;
    for (int o = 1; o < share; o *= 2) rank += __shfl_xor_sync(0xffffffffu, rank, o);
    if (key != 0ull && rank < k && threadIdx.x % share == 0) sh.sorted[rank] = key;
  }
  __syncthreads();
}

// The k best of the n keys held, in order, to sh.sorted and back to the list; returns how many there are.  All threads call it.
__device__ __noinline__ int prune(int n, int k, Shared& sh) {
  const int tid = threadIdx.x;
  if (n > FEW_KEYS) {                                         // first only those that reach a bound of the threads' maxima
    float best = -INFINITY;
    for (int i = tid; i < n; i += NT) best = fmaxf(best, rank_value(sh.keys[i]));
    const float bound = warp_bound(best, k, sh);
    n = compact(n, bound, 0u, 0u, sh);
  }
  rank_keys(sh.keys, n, k, sh);
  const int kept = min(n, k);
  if (tid < kept) sh.keys[tid] = sh.sorted[tid];
  if (tid == 0) sh.n_keys = kept;
  __syncthreads();
  return kept;
}

// AHEAD: the next chunk's columns are on their way while one is worked on (two blocks an SM); else three blocks an SM.
template <typename T, bool RANK, bool TOP, bool AHEAD>
__global__ void __launch_bounds__(NT, AHEAD ? 2 : 3)
token_logprobs_kernel(const T* logits, long ld, int V, const int* tokens, float* __restrict__ logprob, float* __restrict__ entropy,
                      int* __restrict__ rank_out, int top, int* __restrict__ top_ids, float* __restrict__ top_logprobs, int slices) {
  constexpr int VN = Vec<T>::N, NV = PER_THREAD / VN, STEP = NT * NV;
  extern __shared__ __align__(16) unsigned char cluster_raw[];       // a ClusterShared where a cluster shares a row
  __shared__ Shared sh;
  kf_pdl_trigger();
  if (slices > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // waited for before a peer's memory is touched
  kf_pdl_wait();
  logits = kf_produced(logits);                               // no load may stand above the wait
  tokens = kf_produced(tokens);
  const int row = (int)(blockIdx.x / (unsigned)slices), slice = (int)(blockIdx.x % (unsigned)slices);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int token = tokens ? tokens[row] : 0;
  if (token < 0) return;                                      // a row of padding: its whole cluster leaves
  const T* x = logits + (size_t)row * ld;
  const bool inside = token < V;

  // The row: `head` elements up to a 16-byte boundary, `n_vec` vectors, the tail.  Loose elements go to the first slice.
  const int head = min(V, (int)((16 - ((uintptr_t)x & 15)) % 16 / sizeof(T)));
  const int n_vec = (V - head) / VN, loose = V - n_vec * VN;
  const T* body = x + head;
  const int per = (n_vec + slices - 1) / slices;
  const int v_begin = min(n_vec, slice * per), v_end = min(n_vec, v_begin + per);

  auto load = [&](int c, uint4 (&raw)[NV]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = c + j * NT + tid;
      raw[j] = make_uint4(Vec<T>::MASKED, Vec<T>::MASKED, Vec<T>::MASKED, Vec<T>::MASKED);
      if (v < v_end) raw[j] = __ldg(reinterpret_cast<const uint4*>(body) + v);
    }
  };
  uint4 raw[NV];
  load(v_begin, raw);
  const float given = inside ? kf_load(x, token) : 0.f;
  const float given_below = nextafterf(given, -INFINITY);

  Stats st = {-INFINITY, 0.f, 0.f};
  int before = 0;
  const int long_list = 2 * top + 64;                         // a list beyond this is pruned
  float tau = -INFINITY;                                      // what a column must exceed to be a key; masked columns and NaN never are
  if (TOP) {
    if (tid == 0) sh.n_keys = 0;
    __syncthreads();
  }
  if (slice == 0 && tid < loose) {
    const int i = tid < head ? tid : n_vec * VN + tid;
    const float v = kf_load(x, i);
    st.m = v == v ? v : -INFINITY;
    st.s = v == -INFINITY ? 0.f : v == v ? 1.f : v;
    if (RANK) before = (v > given || (v == given && i < token)) ? 1 : 0;
    if (TOP && tid < head && v > tau) sh.keys[atomicAdd(&sh.n_keys, 1)] = rank_key(v, (unsigned)i);
  }

#pragma unroll 1
  for (int c = v_begin; c < v_end; c += STEP) {
    uint4 next[NV];
    if (AHEAD) load(c + STEP, next);                          // (nothing is read beyond the slice)
    else if (c > v_begin) load(c, raw);
    float cm = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VN; ++e) cm = fmaxf(cm, Vec<T>::get(raw[j], e));
    move_to(st, fmaxf(st.m, cm));
    add_exponentials<PER_THREAD>(st, [&](int i) { return Vec<T>::get(raw[i / VN], i % VN); });
    if (RANK) {
      // Columns before the token count when they equal it, columns behind it do not: they must exceed the next lower number, or the
      // token's own.  One by one where the chunk holds the token, ends early (its masked places are no columns) or the token is masked.
      const long i_begin = (long)c * VN + head;
      const bool behind = i_begin > token;
      if (behind || (c + STEP <= v_end && i_begin + CHUNK <= token && given > -INFINITY)) {
        const float over = behind ? given : given_below;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < VN; ++e) before += Vec<T>::get(raw[j], e) > over ? 1 : 0;
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int v = c + j * NT + tid;
          const int earlier = v < v_end ? (int)min((long)VN, (long)token - ((long)v * VN + head)) : 0;       // elements before the token
#pragma unroll
          for (int e = 0; e < VN; ++e) {
            const float value = Vec<T>::get(raw[j], e);
            before += (value > given || (value == given && e < earlier)) ? 1 : 0;
          }
        }
      }
    }
    if (TOP) {
      // Every column above `limit` becomes a key; returns how long the warp saw the list get.  A key that finds the list full is not
      // written, and the length tells.
      auto push = [&](float limit) {
        if (__ballot_sync(0xffffffffu, cm > limit) == 0u) return 0;
        unsigned hits = 0u;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < VN; ++e) hits |= Vec<T>::get(raw[j], e) > limit ? 1u << (j * VN + e) : 0u;
        const int mine = __popc(hits);
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int t = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += t;
        }
        int at = 0;
        if (lane == 31) at = atomicAdd(&sh.n_keys, upto);
        const int seen = __shfl_sync(0xffffffffu, at + upto, 31);
        at = __shfl_sync(0xffffffffu, at, 31) + upto - mine;
        while (hits) {
          const int k = __ffs(hits) - 1;
          hits &= hits - 1;
          const unsigned id = (unsigned)((long)(c + k / VN * NT + tid) * VN + k % VN + head);
          const u64 key = rank_key(pick<T, NV>(raw, k), id);
          if (at < KEY_CAP) sh.keys[at] = key;
          ++at;
        }
        return seen;
      };
      auto settle = [&](int n) {                              // after a prune
        if (n >= top) tau = rank_value(sh.keys[top - 1]);
        __syncthreads();
      };
      float limit = tau;
      bool bounded = false;
      if (c == v_begin) {
        limit = nextafterf(warp_bound(cm, top, sh), -INFINITY);
        bounded = true;
      }
      for (;;) {
        const int seen = push(limit);
        if (!__syncthreads_or(c == v_begin || seen > long_list)) break;
        int n = sh.n_keys;
        __syncthreads();
        if (n <= KEY_CAP) {
          if (n >= top && c + STEP < v_end) settle(prune(n, top, sh));
          break;
        }
        // More than the list holds: the chunk's keys that are in it go, and the chunk comes again, cut by its own bound.
        const unsigned id0 = (unsigned)(c * (long)VN + head), id1 = (unsigned)(min(v_end, c + STEP) * (long)VN + head);
        n = compact(KEY_CAP, -INFINITY, id0, id1, sh);
        if (n >= top) settle(prune(n, top, sh));
        if (!bounded) {
          limit = fmaxf(tau, nextafterf(warp_bound(cm, top, sh), -INFINITY));
          bounded = true;
          continue;
        }
        // Still too many (one value in most places, or most of them masked): one vector of each thread at a time.
#pragma unroll 1
        for (int j = 0; j < NV; ++j) {
          const int v = c + j * NT + tid;
          if (v < v_end)
#pragma unroll 1
            for (int e = 0; e < VN; ++e) {
              const long i = (long)v * VN + e;
              const float value = kf_load(body, i);
              if (value > tau) sh.keys[atomicAdd(&sh.n_keys, 1)] = rank_key(value, (unsigned)(i + head));
            }
          __syncthreads();
          n = sh.n_keys;
          __syncthreads();
          settle(prune(n, top, sh));
        }
        break;
      }
    }
    if (AHEAD) {
#pragma unroll
      for (int j = 0; j < NV; ++j) raw[j] = next[j];
    }
  }

  // The tail's ids are the highest: its keys come last, so that a column that equals tau has a higher id than the key that set it.
  if (TOP && slice == 0 && tid >= head && tid < loose) {
    const int i = n_vec * VN + tid;
    const float v = kf_load(x, i);
    if (v > tau) sh.keys[atomicAdd(&sh.n_keys, 1)] = rank_key(v, (unsigned)i);
  }

  // the block's numbers, then the cluster's
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats other = {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.u, o)};
    join(st, other);
    if (RANK) before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (lane == 0) {
    sh.stats[warp] = st;
    sh.before[warp] = before;
  }
  __syncthreads();
  int n = 0;
  if (TOP) {
    n = sh.n_keys;                                            // within KEY_CAP after every chunk, and the tail
    __syncthreads();
    n = prune(n, top, sh);
  }
  st = sh.stats[0];
  before = sh.before[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) {
    join(st, sh.stats[w]);
    before += sh.before[w];
  }
  if (slices > 1) {
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(cluster_raw);
    uint32_t first;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(first) : "r"(mine));
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");                       // every block of the row has begun
    if (tid == 0) {
      const uint32_t at = first + (uint32_t)offsetof(ClusterShared, stats) + (uint32_t)(sizeof(Stats) * slice);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(st.m) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 4), "f"(st.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 8), "f"(st.u) : "memory");
      asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(first + (uint32_t)offsetof(ClusterShared, before) + 4u * slice), "r"(before) : "memory");
    }
    if (TOP && tid < top)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(first + (uint32_t)offsetof(ClusterShared, keys) + 8u * (slice * top + tid)),
                   "l"(tid < n ? sh.sorted[tid] : 0ull) : "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (slice != 0) return;
    const ClusterShared& all = *reinterpret_cast<const ClusterShared*>(cluster_raw);
    st = all.stats[0];
    before = all.before[0];
    for (int r = 1; r < slices; ++r) {
      join(st, all.stats[r]);
      before += all.before[r];
    }
    if (TOP) {
      // The lists are in order: at least `top` of their keys reach the smallest of the lists' q-th keys, q = ceil(top / slices).
      const int q = (top + slices - 1) / slices;
      u64 bound = all.keys[q - 1];
      for (int r = 1; r < slices; ++r) bound = min(bound, all.keys[r * top + q - 1]);
      if (tid == 0) sh.n_keys = 0;
      __syncthreads();
      for (int i = tid; i < slices * top; i += NT) {
        const u64 key = all.keys[i];
        if (key != 0ull && key >= bound) sh.keys[atomicAdd(&sh.n_keys, 1)] = key;
      }
      __syncthreads();
      n = sh.n_keys;
      rank_keys(sh.keys, n, top, sh);
    }
  }
  if (TOP && n < top) {
    // Fewer columns above -inf than alternatives: the first masked ones follow, then NaN, each in order of their ids.
    if (warp == 0)
      for (int kind = 0; kind < 2; ++kind)
        for (int i0 = 0; i0 < V && n < top; i0 += 32) {
          const float v = i0 + lane < V ? kf_load(x, i0 + lane) : 0.f;
          const bool hit = i0 + lane < V && (kind == 0 ? v == -INFINITY : v != v);
          const unsigned hits = __ballot_sync(0xffffffffu, hit);
          const int at = n + __popc(hits & ((1u << lane) - 1u));
          if (hit && at < top) sh.sorted[at] = rank_key(v, (unsigned)(i0 + lane));
          n += __popc(hits);
        }
    __syncthreads();
  }
  if (tid == 0) {
    if (logprob) logprob[row] = row_logprob(st, inside ? given : __int_as_float(0x7fffffff));
    if (entropy) entropy[row] = row_entropy(st);
    if (RANK) rank_out[row] = inside && given == given ? before : -1;
  }
  if (TOP && tid < top) {
    const u64 key = sh.sorted[tid];
    if (top_ids) top_ids[(size_t)row * top + tid] = rank_id(key);
    if (top_logprobs) top_logprobs[(size_t)row * top + tid] = row_logprob(st, rank_value(key));
  }
}

template <typename T, bool RANK, bool TOP, bool AHEAD>
int launch(const void* logits, long ld, int R, int V, const int* tokens, float* logprob, float* entropy, int* rank, int top,
           int* top_ids, float* top_logprobs, int slices, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)R * (unsigned)slices);
  cfg.blockDim = dim3(NT);
  cfg.stream = stream;
  cfg.dynamicSmemBytes = slices > 1 ? sizeof(ClusterShared) : 0;
  if (slices > 8) {
    static bool allowed[64] = {};                             // by device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !allowed[dev]) {
      if (cudaFuncSetAttribute(token_logprobs_kernel<T, RANK, TOP, AHEAD>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
        kf_record_cuda_error(cudaGetLastError());
        return KF_ERR_SETUP;
      }
      if (dev >= 0 && dev < 64) allowed[dev] = true;
    }
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)slices;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kf_pdl_enabled() ? 2 : 1;
  cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, RANK, TOP, AHEAD>, (const T*)logits, ld, V, tokens, logprob, entropy, rank, top, top_ids,
                     top_logprobs, slices);
  KF_CHECK_LAUNCH();
  return KF_OK;
}

template <typename T, bool AHEAD>
int launch_type(const void* logits, long ld, int R, int V, const int* tokens, float* logprob, float* entropy, int* rank, int top,
                int* top_ids, float* top_logprobs, int slices, cudaStream_t stream) {
  const auto f = rank ? (top ? launch<T, true, true, AHEAD> : launch<T, true, false, AHEAD>)
                      : (top ? launch<T, false, true, AHEAD> : launch<T, false, false, AHEAD>);
  return f(logits, ld, R, V, tokens, logprob, entropy, rank, top, top_ids, top_logprobs, slices, stream);
}

}  // namespace

// logits [R, V] of element type dt (KF_F32, KF_BF16), rows ld elements apart; tokens [R] (null: only entropy and alternatives;
// a negative one: the row's outputs stay as they are; one >= V, or one whose logit is NaN: NaN and rank -1); every output may be null; top <= 64, <= V.
KF_API int kf_token_logprobs(const void* logits, int dt, long ld, int R, int V, const int* tokens, float* logprob, float* entropy,
                             int* rank, int top, int* top_ids, float* top_logprobs, cudaStream_t stream) {
  if (R <= 0) return KF_OK;
  if (V <= 0 || V > 0x7fffff00 || R > (1 << 27) || top < 0 || top > TOP_MAX || top > V || (!tokens && (logprob || rank))) return KF_ERR_SIZE;
  if (((uintptr_t)logits & (dt == KF_F32 ? 3 : 1)) != 0) return KF_ERR_ALIGN;
  // A row is cut while its slices still fit the device at once (two blocks an SM) and each is more than half a chunk.  32-bit logits, L2
  // flushed, slices 1 / 2 / 4 / 8 / 16: 64 x 256,000 with 20 alternatives 49 / 35 / 31 / 39 / 56 us, 8 x 256,000 47 / 32 / 23 / 18 / 18,
  // 512 x 256,000 132 / 139 / 174 / 228 / 339, 301 x 32,003 28 / 35 / 43 / 74 / 142.
  const int chunks = kf_ceil_div(V, CHUNK);
  int slices = 1;
  while (slices < MAX_SLICES && slices < chunks && (long)R * slices <= kf_sm_count()) slices *= 2;
  // Rows of a few chunks that need more than two blocks an SM: a block's start and end are most of its time, and a third block hides more of
  // them than loads ahead do.  2,048 x 32,000 with 20 alternatives 100 us ahead, 92 not, without alternatives 57 and 54; 301 x 32,003 with
  // 64 alternatives 38 and 35; 512 x 256,000 89 and 115.
  const bool ahead = kf_ceil_div(chunks, slices) > 4 || (long)R * slices <= 2l * kf_sm_count();
  if (dt != KF_F32 && dt != KF_BF16) return KF_ERR_DTYPE;
  const auto f = dt == KF_F32 ? (ahead ? launch_type<float, true> : launch_type<float, false>)
                              : (ahead ? launch_type<__nv_bfloat16, true> : launch_type<__nv_bfloat16, false>);
  return f(logits, ld, R, V, tokens, logprob, entropy, rank, top, top_ids, top_logprobs, slices, stream);
}
