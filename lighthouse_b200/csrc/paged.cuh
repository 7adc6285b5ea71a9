// Attention of new tokens over a paged key-value cache: what its kernels share. The keys of a
// sequence are cut into tiles; all tiles of a call form one line (sequence, then unit, then
// tile; a unit is a kv head and a group of its query rows), and every CTA takes an equal
// stretch of that line. The lengths live on the device, so each CTA works out its stretch
// itself: a call needs no knowledge of them on the host, replays as a graph while sequences
// grow, and a ragged batch is balanced to within one tile.
#pragma once
#include "common.cuh"
#include "epilogue.cuh"
#include "ptx.cuh"

namespace lh {

__device__ __forceinline__ void report_bad_index(int* dev_status) { atomicCAS(dev_status, 0, DEV_BAD_INDEX); }

struct PagedParams {
  const void* q; const void* k; const void* v; void* o;
  int64_t sqb, sqh, sqs;  // unit stride in the head dimension everywhere
  int64_t sob, soh, sos;
  int64_t skp, sks, skh;
  int64_t svp, svs, svh;
  const int* table; int64_t stb, stp;
  const int* lengths; int64_t slen;
  int64_t num_pages;
  int B, Hkv, group, Sq, D;
  int page, page_shift;   // page_shift < 0: the page size is no power of two
  int max_keys;           // table columns x page size
  int rows, unit_rows, row_groups;  // query rows of a kv head (tokens x group), rows of a unit, units of a kv head
  int tile;               // keys of a tile
  int o_dtype;
  float scale_log2;       // softmax scale x log2(e): scores are kept as powers of two
  // workspace
  int64_t* total;         // tiles of the whole call
  int4* first;            // per CTA: (sequence, unit, tile) its stretch starts at; x < 0: no stretch
  float2* ml;             // per partial row: running maximum and sum
  float* part;            // per partial row: Dp floats, not yet divided by the sum
  int Dp;
  int* dev_status;
};

// CTA i of n owns tiles [total * i / n, total * (i + 1) / n); no stretch is empty because n <= total.
__host__ __device__ __forceinline__ int64_t stretch_begin(int64_t total, int64_t n, int64_t i) { return total * i / n; }
// The CTA that owns tile x: the last i with total * i / n < x + 1.
__host__ __device__ __forceinline__ int64_t stretch_owner(int64_t total, int64_t n, int64_t x) { return ((x + 1) * n - 1) / total; }

__device__ __forceinline__ int paged_length(const PagedParams& p, int b) {
  const int len = p.lengths[b * p.slen];
  return len < 0 ? 0 : len > p.max_keys ? p.max_keys : len;
}
__device__ __forceinline__ int paged_tiles(const PagedParams& p, int len) { return (len + p.tile - 1) / p.tile; }

__device__ __forceinline__ int page_of(const PagedParams& p, int j) { return p.page_shift >= 0 ? j >> p.page_shift : j / p.page; }

// A position on the line of tiles.
struct TileCursor {
  int b, u, t, tiles, len;
  __device__ __forceinline__ void seek(const PagedParams& p, int b_, int64_t within) {
    b = b_;
    len = paged_length(p, b);
    tiles = paged_tiles(p, len);
    u = static_cast<int>(within / tiles);
    t = static_cast<int>(within % tiles);
  }
  // Only called while tiles of this CTA's stretch remain, so the next sequence exists.
  __device__ __forceinline__ void next_unit(const PagedParams& p) {
    t = 0;
    if (++u < p.Hkv * p.row_groups) return;
    u = 0;
    do {
      ++b;
      len = paged_length(p, b);
    } while (len == 0);
    tiles = paged_tiles(p, len);
  }
};

// Every thread of the block gets this CTA's stretch [lo, hi) and where it starts.
// Prefix sum over the sequences: each thread adds up a run of them, the block scans the runs.
template <int NT>
__device__ __forceinline__ bool find_stretch(const PagedParams& p, int64_t& lo, int64_t& hi, TileCursor& at) {
  __shared__ int64_t warp_sum[NT / 32];
  __shared__ int64_t start_base;
  __shared__ int start_b;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int units = p.Hkv * p.row_groups;
  const int run = (p.B + NT - 1) / NT;
  const int64_t first = static_cast<int64_t>(tid) * run;  // B can be near 2^31
  const int b0 = first < p.B ? static_cast<int>(first) : p.B;
  const int b1 = first + run < p.B ? static_cast<int>(first + run) : p.B;
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    const int raw = p.lengths[b * p.slen];
    if (blockIdx.x == 0 && (raw < 0 || raw > p.max_keys)) report_bad_index(p.dev_status);
    mine += static_cast<int64_t>(paged_tiles(p, paged_length(p, b))) * units;
  }
  int64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  const int64_t n = total < gridDim.x ? total : gridDim.x;
  if (blockIdx.x == 0 && tid == 0) *p.total = total;
  if (blockIdx.x >= n) {
    if (tid == 0) p.first[blockIdx.x] = make_int4(-1, 0, 0, 0);
    return false;
  }
  lo = stretch_begin(total, n, blockIdx.x);
  hi = stretch_begin(total, n, blockIdx.x + 1);
  int64_t base = before + incl - mine;
  if (lo >= base && lo < base + mine) {
    for (int b = b0; b < b1; ++b) {
      const int64_t here = static_cast<int64_t>(paged_tiles(p, paged_length(p, b))) * units;
      if (lo < base + here) {
        start_b = b;
        start_base = base;
        break;
      }
      base += here;
    }
  }
  __syncthreads();
  at.seek(p, start_b, lo - start_base);
  if (tid == 0) p.first[blockIdx.x] = make_int4(at.b, at.u, at.t, 0);
  return true;
}

// Where this CTA's part of unit (tiles t0 .. t1 of `tiles`) goes: -1 when it is the whole unit,
// else one of the CTA's two partial slots (the stretch's first unit may begin before it, its
// last may end after it).
__device__ __forceinline__ int64_t partial_slot(int t0, int t1, int tiles) {
  if (t0 == 0 && t1 == tiles) return -1;
  return 2 * static_cast<int64_t>(blockIdx.x) + (t0 == 0 ? 1 : 0);
}

// 2^(x - m) against a running maximum m. Before any key counted (m = -inf) a score is either
// -inf, of no weight, or NaN, which stays one.
__device__ __forceinline__ float exp2_safe(float x, float m) { return m == -INFINITY ? (x == -INFINITY ? 0.f : x) : exp2f(x - m); }

// Query row r of unit u: which token and head it is.
__device__ __forceinline__ int row_token(const PagedParams& p, int row) { return row / p.group; }
__device__ __forceinline__ int row_head(const PagedParams& p, int hkv, int row) { return hkv * p.group + row % p.group; }

// The tensor-core kernel (paged_mma.cu).
bool paged_mma_supported(const lh_memref_t* k, const lh_memref_t* v);
int paged_mma_unit_rows(int64_t rows, int D);
int paged_mma_ctas(const lh_ctx* ctx, int D);
int paged_mma_launch(lh_ctx* ctx, PagedParams& p, int dtype, int ctas);

}  // namespace lh
