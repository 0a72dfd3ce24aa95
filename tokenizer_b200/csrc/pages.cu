// Copies of cache pages: what a fork of requests moves.  A fork shares the full pages of its parent and gets a copy of the
// last, partly filled one, in every plane (layer, keys or values) of the pool.
//
// The pool is [planes][pages][page bytes]; a pair (source, destination, rows) copies the first `rows` rows of a page, which
// lie side by side, so a copy is one run of bytes a plane.  The pairs travel in the launch's arguments: no copy to the
// device in front of the kernel, and a captured launch keeps them.  63 copies in 56 planes of a large model: 7.7 us on the
// device (floor 4.5), 3 copies in 48 planes 1.5.
#include "common.cuh"

#define PC_PAIRS 256           // pairs of one launch: 3 KB of arguments
#define PC_THREADS 256
#define PC_PIECES 4            // words of a thread, asked for before the first is stored

struct PagePairs { int source[PC_PAIRS], target[PC_PAIRS], rows[PC_PAIRS]; };

template <typename Word>
__global__ void __launch_bounds__(PC_THREADS)
copy_pages_kernel(Word* __restrict__ pool, long long plane_words, long long page_words, int row_words,
                  const __grid_constant__ PagePairs pairs) {
  pdl_wait();
  pdl_launch();
  const int pair = blockIdx.y;
  const long long words = (long long)pairs.rows[pair] * row_words;
  Word* plane = pool + blockIdx.z * plane_words;
  const Word* from = plane + pairs.source[pair] * page_words;
  Word* to = plane + pairs.target[pair] * page_words;
  for (long long at = (long long)blockIdx.x * (PC_THREADS * PC_PIECES) + threadIdx.x; at < words;
       at += (long long)gridDim.x * (PC_THREADS * PC_PIECES)) {
    Word held[PC_PIECES];
#pragma unroll
    for (int i = 0; i < PC_PIECES; ++i)
      if (at + i * PC_THREADS < words) held[i] = from[at + i * PC_THREADS];
#pragma unroll
    for (int i = 0; i < PC_PIECES; ++i)
      if (at + i * PC_THREADS < words) to[at + i * PC_THREADS] = held[i];
  }
}

// Whether the pairs can be copied in any order: pages of the pool, rows of a page, no destination twice and none that is
// also a source.
static int pairs_status(const int* flat, int n, long long pages, int page) {
  if (pages > 0x7fffffffLL) return TOKB200_BAD_SIZE;
  unsigned char* written = (unsigned char*)calloc((size_t)(pages / 8 + 1), 1);
  if (!written) return TOKB200_BAD_SIZE;
  int status = TOKB200_OK;
  for (int i = 0; i < n && status == TOKB200_OK; ++i) {
    const int source = flat[3 * i], target = flat[3 * i + 1], rows = flat[3 * i + 2];
    if (source < 0 || source >= pages || target < 0 || target >= pages || rows < 0 || rows > page ||
        (written[target / 8] >> (target % 8) & 1))
      status = TOKB200_BAD_SIZE;
    else
      written[target / 8] |= (unsigned char)(1 << (target % 8));
  }
  for (int i = 0; i < n && status == TOKB200_OK; ++i)
    if (written[flat[3 * i] / 8] >> (flat[3 * i] % 8) & 1) status = TOKB200_BAD_SIZE;
  free(written);
  return status;
}

// The checks alone, for callers without a GPU.
TOKB200_API int tokb200_copy_pages_check(const int* flat, int n, long long pages, int page) {
  return n < 0 || page <= 0 || pages < 0 ? TOKB200_BAD_SIZE : pairs_status(flat, n, pages, page);
}

// `flat`: n (source, destination, rows) on the host; the pool has `planes` planes of `pages` pages of `page` rows of
// `row_bytes` each.
TOKB200_API int tokb200_copy_pages(void* pool, int planes, long long pages, int page, long long row_bytes, const int* flat, int n,
                                   cudaStream_t stream) {
  if (planes <= 0 || planes > 65535 || page <= 0 || pages < 0 || row_bytes <= 0 || row_bytes > 0x7fffffffLL || n < 0)
    return TOKB200_BAD_SIZE;
  int status = pairs_status(flat, n, pages, page);
  // the widest word that a row is a whole number of and the pool is aligned to
  const unsigned long long odd = (unsigned long long)(uintptr_t)pool | (unsigned long long)row_bytes;
  const int word = odd % 16 == 0 ? 16 : odd % 4 == 0 ? 4 : odd % 2 == 0 ? 2 : 1;
  const int row_words = (int)(row_bytes / word);
  const long long page_words = (long long)row_words * page, plane_words = page_words * pages;
  for (int first = 0; first < n && status == TOKB200_OK; first += PC_PAIRS) {
    const int here = n - first < PC_PAIRS ? n - first : PC_PAIRS;
    PagePairs pairs;
    long long most = 0;
    for (int i = 0; i < PC_PAIRS; ++i) {
      const int* p = flat + 3 * (first + i);
      pairs.source[i] = i < here ? p[0] : 0;
      pairs.target[i] = i < here ? p[1] : 0;
      pairs.rows[i] = i < here ? p[2] : 0;
      if (pairs.rows[i] > most) most = pairs.rows[i];
    }
    if (most == 0) continue;
    const long long pieces = (most * row_words + PC_THREADS * PC_PIECES - 1) / (PC_THREADS * PC_PIECES);
    const dim3 grid((unsigned)(pieces < 65535 ? pieces : 65535), here, planes);
    if (word == 16)
      status = launch_dependent(copy_pages_kernel<uint4>, grid, dim3(PC_THREADS), 0, stream, (uint4*)pool, plane_words, page_words, row_words, pairs);
    else if (word == 4)
      status = launch_dependent(copy_pages_kernel<unsigned>, grid, dim3(PC_THREADS), 0, stream, (unsigned*)pool, plane_words, page_words, row_words, pairs);
    else if (word == 2)
      status = launch_dependent(copy_pages_kernel<unsigned short>, grid, dim3(PC_THREADS), 0, stream, (unsigned short*)pool, plane_words, page_words, row_words, pairs);
    else
      status = launch_dependent(copy_pages_kernel<unsigned char>, grid, dim3(PC_THREADS), 0, stream, (unsigned char*)pool, plane_words, page_words, row_words, pairs);
  }
  return status;
}
