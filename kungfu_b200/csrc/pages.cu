// Pages of a cache (or rows of per-request states) copied in every store of the cache by one launch: store s is an array of
// pages of bytes[s] bytes, and page src[i] becomes page dst[i] of the same store.  No destination is a source and none occurs
// twice (the caller checks), so the copies are independent of one another.
#include "common.cuh"

namespace {

constexpr int MAX_STORES = 64, MAX_PAIRS = 256;

// Everything the host knows travels as the kernel's own argument (3.1 KB): no table to allocate, copy in or keep alive.
struct PageCopies {
  char* base[MAX_STORES];
  long bytes[MAX_STORES];
  int src[MAX_PAIRS], dst[MAX_PAIRS];
};

// One block copies one page of one store, in units of U (the widest that the page's size and the store's address allow).
template <typename U>
__device__ __forceinline__ void copy_units(const char* from, char* to, long n) {
  for (long i = threadIdx.x; i < n; i += blockDim.x) reinterpret_cast<U*>(to)[i] = reinterpret_cast<const U*>(from)[i];
}

__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ PageCopies c) {
  kf_pdl_trigger();
  kf_pdl_wait();
  const int pair = blockIdx.x, store = blockIdx.y;
  const long bytes = c.bytes[store];
  const char* from = c.base[store] + (size_t)c.src[pair] * bytes;
  char* to = c.base[store] + (size_t)c.dst[pair] * bytes;
  const unsigned long align = (unsigned long)c.base[store] | (unsigned long)bytes;
  if (align % 16 == 0) copy_units<int4>(from, to, bytes / 16);
  else if (align % 4 == 0) copy_units<int>(from, to, bytes / 4);
  else if (align % 2 == 0) copy_units<short>(from, to, bytes / 2);
  else copy_units<char>(from, to, bytes);
}

}  // namespace

KF_API int kf_copy_pages_max_stores() { return MAX_STORES; }
KF_API int kf_copy_pages_max_pairs() { return MAX_PAIRS; }

// bases, bytes [n_stores <= 64], src, dst [n_pairs <= 256]: host arrays.
KF_API int kf_copy_pages(const int64_t* bases, const int64_t* bytes, int n_stores, const int* src, const int* dst, int n_pairs,
                         cudaStream_t stream) {
  if (n_stores <= 0 || n_pairs <= 0) return KF_OK;
  if (n_stores > MAX_STORES || n_pairs > MAX_PAIRS) return KF_ERR_SIZE;
  PageCopies c;
  for (int s = 0; s < n_stores; ++s) {
    c.base[s] = (char*)bases[s];
    c.bytes[s] = (long)bytes[s];
  }
  for (int i = 0; i < n_pairs; ++i) {
    c.src[i] = src[i];
    c.dst[i] = dst[i];
  }
  kf_launch(copy_pages_kernel, dim3(n_pairs, n_stores), dim3(256), 0, stream, c);
  KF_CHECK_LAUNCH();
  return KF_OK;
}
