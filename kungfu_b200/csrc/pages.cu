// Pages of a cache (or rows of per-request states) copied in every store of the cache by one launch: store s is an array of
// pages of bytes[s] bytes, and page src[i] becomes page dst[i] of the same store.  No destination is a source and none occurs
// twice (the caller checks), so the copies are independent of one another.
//
// Bound by memory.  A block copies one piece of one page: 8 units of 16 bytes a thread, all on their way before the first is
// stored (32 KB a block, several blocks an SM: more in flight than memory's latency takes).  Pages whose size or address is no multiple of
// 16 bytes start at another phase each, so they go in the widest unit that their store allows, 16 a thread.  8 stores x 256 pages of
// 128 KB in 82 us (6.55 TB/s read and written, as fast as one plain copy of as much); 4-byte units 5.9 TB/s, 2-byte units 4.4.
#include "common.cuh"

namespace {

constexpr int MAX_STORES = 64, MAX_PAIRS = 256;

// Everything the host knows travels as the kernel's own argument (3.6 KB): no table to allocate, copy in or keep alive.
struct PageCopies {
  char* base[MAX_STORES];
  long bytes[MAX_STORES];
  unsigned first[MAX_STORES];                                   // the first block of each store
  int unit[MAX_STORES];                                         // 16, 4, 2 or 1 bytes
  int src[MAX_PAIRS], dst[MAX_PAIRS];
  int n_stores, n_pairs;
};
constexpr int CP_THREADS = 256;
__host__ __device__ constexpr int units_per_thread(int unit) { return unit == 16 ? 8 : 16; }
__host__ __device__ constexpr int piece_bytes(int unit) { return CP_THREADS * units_per_thread(unit) * unit; }

template <typename U>
__device__ __forceinline__ void copy_piece(const char* from, char* to, long bytes, long piece) {
  constexpr int N = units_per_thread(sizeof(U));
  const long i0 = piece * (CP_THREADS * N) + threadIdx.x, n = bytes / (long)sizeof(U);
  U held[N];
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (i0 + j * CP_THREADS < n) held[j] = __ldcs(reinterpret_cast<const U*>(from) + i0 + j * CP_THREADS);
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (i0 + j * CP_THREADS < n) __stcs(reinterpret_cast<U*>(to) + i0 + j * CP_THREADS, held[j]);
}

__global__ void __launch_bounds__(CP_THREADS) copy_pages_kernel(const __grid_constant__ PageCopies c) {
  kf_pdl_trigger();
  int s = 0;
  for (int step = MAX_STORES / 2; step > 0; step /= 2)
    if (s + step < c.n_stores && c.first[s + step] <= blockIdx.x) s += step;
  const unsigned in_store = blockIdx.x - c.first[s];
  const int pair = (int)(in_store % (unsigned)c.n_pairs);
  const long piece = in_store / (unsigned)c.n_pairs, bytes = c.bytes[s];
  const char* from = c.base[s] + (size_t)c.src[pair] * bytes;
  char* to = c.base[s] + (size_t)c.dst[pair] * bytes;
  kf_pdl_wait();
  if (c.unit[s] == 16) copy_piece<int4>(from, to, bytes, piece);
  else if (c.unit[s] == 4) copy_piece<int>(from, to, bytes, piece);
  else if (c.unit[s] == 2) copy_piece<short>(from, to, bytes, piece);
  else copy_piece<signed char>(from, to, bytes, piece);
}

}  // namespace

// bases, bytes [n_stores <= 64], src, dst [n_pairs <= 256]: host arrays.
KF_API int kf_copy_pages(const int64_t* bases, const int64_t* bytes, int n_stores, const int* src, const int* dst, int n_pairs,
                         cudaStream_t stream) {
  if (n_stores <= 0 || n_pairs <= 0) return KF_OK;
  if (n_stores > MAX_STORES || n_pairs > MAX_PAIRS) return KF_ERR_SIZE;
  PageCopies c;
  c.n_stores = n_stores;
  c.n_pairs = n_pairs;
  long blocks = 0;
  for (int s = 0; s < n_stores; ++s) {
    const unsigned long align = (unsigned long)bases[s] | (unsigned long)bytes[s];
    c.base[s] = (char*)bases[s];
    c.bytes[s] = (long)bytes[s];
    c.unit[s] = align % 16 == 0 ? 16 : align % 4 == 0 ? 4 : align % 2 == 0 ? 2 : 1;
    c.first[s] = (unsigned)blocks;
    const long piece = piece_bytes(c.unit[s]);
    blocks += (c.bytes[s] + piece - 1) / piece * n_pairs;
    if (blocks > 0x7fffffffl) return KF_ERR_SIZE;
  }
  for (int i = 0; i < n_pairs; ++i) {
    c.src[i] = src[i];
    c.dst[i] = dst[i];
  }
  kf_launch(copy_pages_kernel, dim3((unsigned)blocks), dim3(CP_THREADS), 0, stream, c);
  KF_CHECK_LAUNCH();
  return KF_OK;
}
