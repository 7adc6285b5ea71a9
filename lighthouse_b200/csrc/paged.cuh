// Attention of new tokens over a paged key-value cache: what its kernels share. The keys of a
// sequence are cut into tiles of 16; all tiles of a call form one line (sequence, then unit, then
// tile; a unit is a kv head and a group of its query rows), and every WARP takes an equal stretch
// of that line, with loads, online softmax and results of its own. A unit costs its warp some tiles' time
// besides its tiles (Q, the epilogue), so the line counts that too: a unit takes unit_cost places and
// then one per tile, and a stretch that would begin within the former begins with the unit. The
// lengths live on the device, so each CTA works out its warps' stretches itself: a call needs
// no knowledge of them on the host, replays as a graph while sequences grow, and a ragged batch
// is balanced. Where a stretch ends inside a unit, the warp leaves a partial result to the join
// kernel.
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
  int unit_cost;          // places on the line that a unit takes besides its tiles
  int o_dtype, o_vec;     // o_vec: four elements of a row of o can be stored at once
  int q_pairs;            // two 16-bit elements of a row of q can be loaded at once
  float scale_log2;       // softmax scale x log2(e): scores are kept as powers of two
  // workspace
  int64_t* total;         // length of the line
  int4* first;            // per stretch: (sequence, unit, tile) it starts at and the unit's tiles; x < 0: it has none
  float2* ml;             // per partial row: running maximum and sum
  float* part;            // per partial row: Dp floats, not yet divided by the sum
  int Dp, part_rows;      // floats of a partial row, rows of a partial result
  int* dev_status;
};

constexpr int TILE = 16;  // keys of a tile
constexpr int JOIN_WARPS = 8;

// How many stretches a line of `total` places is cut into. Shorter ones than two places would only give
// the join more parts: one sequence of 7117 keys on four kv heads takes 28.6 us cut into single places, 22.6 so
// (22.5 with three; with four and more a tile after the other begins to cost, 129 keys 16.4 -> 18.4).
constexpr int SHORTEST = 2;
__host__ __device__ __forceinline__ int64_t stretch_count(int64_t total, int64_t warps) {
  const int64_t n = (total + SHORTEST - 1) / SHORTEST;
  return n < warps ? n : warps;
}

// Stretch i of n is places [total * i / n, total * (i + 1) / n) of the line; n <= total.
// (n is some thousands at most, so 32-bit division serves all but the longest calls in a quarter of the time.)
__host__ __device__ __forceinline__ int64_t stretch_begin(int64_t total, int64_t n, int64_t i) {
  const int64_t x = total * i;
  return x < 0x7fffffff ? static_cast<int64_t>(static_cast<uint32_t>(x) / static_cast<uint32_t>(n)) : x / n;
}
// The stretch that has place x: the last i with total * i / n < x + 1.
__host__ __device__ __forceinline__ int64_t stretch_owner(int64_t total, int64_t n, int64_t x) {
  const int64_t y = (x + 1) * n - 1;
  return y < 0x7fffffff ? static_cast<int64_t>(static_cast<uint32_t>(y) / static_cast<uint32_t>(total)) : y / total;
}

__device__ __forceinline__ int paged_length(const PagedParams& p, int b) {
  const int len = p.lengths[b * p.slen];
  return len < 0 ? 0 : len > p.max_keys ? p.max_keys : len;
}
__device__ __forceinline__ int paged_tiles(int len) { return (len + TILE - 1) / TILE; }

__device__ __forceinline__ int page_of(const PagedParams& p, int j) { return p.page_shift >= 0 ? j >> p.page_shift : j / p.page; }

// A position on the line of tiles.
struct TileCursor {
  int b, u, t, tiles, len;
  // `within`: places from the sequence's first on.
  __device__ __forceinline__ void seek(const PagedParams& p, int b_, int64_t within) {
    b = b_;
    len = paged_length(p, b);
    tiles = paged_tiles(len);
    const int unit = tiles + p.unit_cost;
    u = within < 0x7fffffff ? static_cast<int>(static_cast<uint32_t>(within) / static_cast<uint32_t>(unit)) : static_cast<int>(within / unit);
    t = max(0, static_cast<int>(within - static_cast<int64_t>(u) * unit) - p.unit_cost);
  }
  // Only called while tiles of this warp's stretch remain, so the next sequence exists.
  __device__ __forceinline__ void next_unit(const PagedParams& p) {
    t = 0;
    if (++u < p.Hkv * p.row_groups) return;
    u = 0;
    do {
      ++b;
      len = paged_length(p, b);
    } while (len == 0);
    tiles = paged_tiles(len);
  }
};

// Each warp learns how many tiles its stretch has and where it starts; 0 for warps without any. Prefix
// sums over the sequences: each thread adds up a run of them, the block scans the runs. All
// threads call it.
template <int NT>
__device__ __forceinline__ int64_t find_stretch(const PagedParams& p, TileCursor& at) {
  constexpr int W = NT / 32;
  __shared__ int64_t warp_places[W], warp_tiles[W];
  __shared__ int64_t start_places[W + 1], start_tiles[W + 1];  // of the sequence that each border lies in: places from its first on, tiles before it
  __shared__ int start_b[W + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int units = p.Hkv * p.row_groups;
  const int run = (p.B + NT - 1) / NT;
  const int64_t first = static_cast<int64_t>(tid) * run;  // B can be near 2^31
  const int b0 = first < p.B ? static_cast<int>(first) : p.B;
  const int b1 = first + run < p.B ? static_cast<int>(first + run) : p.B;
  auto tiles_of = [&](int b) { return paged_tiles(paged_length(p, b)); };
  auto places_of = [&](int tiles) { return tiles ? static_cast<int64_t>(tiles + p.unit_cost) * units : 0; };
  int64_t my_places = 0, my_tiles = 0;
  for (int b = b0; b < b1; ++b) {
    const int raw = p.lengths[b * p.slen];
    if (blockIdx.x == 0 && (raw < 0 || raw > p.max_keys)) report_bad_index(p.dev_status);
    const int tiles = tiles_of(b);
    my_places += places_of(tiles);
    my_tiles += static_cast<int64_t>(tiles) * units;
  }
  int64_t places = my_places, tiles_incl = my_tiles;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, places, d), up_t = __shfl_up_sync(0xffffffffu, tiles_incl, d);
    if (lane >= d) {
      places += up;
      tiles_incl += up_t;
    }
  }
  if (lane == 31) {
    warp_places[warp] = places;
    warp_tiles[warp] = tiles_incl;
  }
  __syncthreads();
  int64_t total = 0, all_tiles = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) {
      places += warp_places[w];
      tiles_incl += warp_tiles[w];
    }
    total += warp_places[w];
    all_tiles += warp_tiles[w];
  }
  const int64_t stretches = static_cast<int64_t>(gridDim.x) * W;
  const int64_t n = stretch_count(total, stretches);
  if (blockIdx.x == 0 && tid == 0) *p.total = total;
  const int64_t base = places - my_places;
  for (int w = 0; w <= W; ++w) {  // the CTA's borders: where each warp's stretch begins, and the last one's ends
    const int64_t s = static_cast<int64_t>(blockIdx.x) * W + w;
    if (s >= n) break;
    const int64_t begin = stretch_begin(total, n, s);
    if (begin < base || begin >= places) continue;
    int64_t at_place = base, at_tile = tiles_incl - my_tiles;
    for (int b = b0; b < b1; ++b) {
      const int tiles = tiles_of(b);
      const int64_t here = places_of(tiles);
      if (begin < at_place + here) {
        start_b[w] = b;
        start_places[w] = begin - at_place;
        start_tiles[w] = at_tile;
        break;
      }
      at_place += here;
      at_tile += static_cast<int64_t>(tiles) * units;
    }
  }
  __syncthreads();
  const int64_t s = static_cast<int64_t>(blockIdx.x) * W + warp;
  int64_t left = 0;
  if (s < n) {
    int64_t end = all_tiles;
    if (s + 1 < n) {
      TileCursor to;
      to.seek(p, start_b[warp + 1], start_places[warp + 1]);
      end = start_tiles[warp + 1] + static_cast<int64_t>(to.u) * to.tiles + to.t;
    }
    at.seek(p, start_b[warp], start_places[warp]);
    left = end - (start_tiles[warp] + static_cast<int64_t>(at.u) * at.tiles + at.t);
  }
  if (lane == 0) p.first[s] = left ? make_int4(at.b, at.u, at.t, at.tiles) : make_int4(-1, 0, 0, 0);
  return left;
}

// Where a warp's part of a unit (tiles t0 .. t1 of `tiles`) goes: -1 when it is the whole unit, else
// one of the stretch's two partial slots (its first unit may begin before it, its last may end
// after it).
template <int NT>
__device__ __forceinline__ int64_t partial_slot(int t0, int t1, int tiles) {
  if (t0 == 0 && t1 == tiles) return -1;
  return 2 * (static_cast<int64_t>(blockIdx.x) * (NT / 32) + (threadIdx.x >> 5)) + (t0 == 0 ? 1 : 0);
}

// 2^(x - m) against a running maximum m. Before any key counted (m = -inf) a score is either
// -inf, of no weight, or NaN, which stays one.
__device__ __forceinline__ float exp2_safe(float x, float m) { return m == -INFINITY ? (x == -INFINITY ? 0.f : x) : exp2f(x - m); }

// Four head dimensions from d on of a row of o (those below D).
__device__ __forceinline__ void store_o4(const PagedParams& p, int64_t row, int d, float4 v) {
  if (p.o_vec) {  // D is a multiple of four
    if (d >= p.D) return;
    if (p.o_dtype == LH_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p.o) + row + d) = v;
    } else if (p.o_dtype == LH_BF16) {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.o) + row + d) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
      const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
      *reinterpret_cast<uint2*>(static_cast<__half*>(p.o) + row + d) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
    return;
  }
  if (d < p.D) store_from_f32(p.o, p.o_dtype, row + d, v.x);
  if (d + 1 < p.D) store_from_f32(p.o, p.o_dtype, row + d + 1, v.y);
  if (d + 2 < p.D) store_from_f32(p.o, p.o_dtype, row + d + 2, v.z);
  if (d + 3 < p.D) store_from_f32(p.o, p.o_dtype, row + d + 3, v.w);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// What the side of a warp that fetches knows: the next tile to fetch and, one step ahead of its use,
// the page that holds this lane's key of it.
struct Fetch {
  TileCursor at;
  int64_t left;  // tiles still to fetch
  int page_id;
  __device__ __forceinline__ void look_up(const PagedParams& p, int key_in_tile) {
    const int j = at.t * TILE + key_in_tile;
    page_id = left > 0 && j < at.len ? p.table[at.b * p.stb + page_of(p, j) * p.stp] : -1;
  }
  __device__ __forceinline__ void advance(const PagedParams& p) {
    --left;
    if (++at.t == at.tiles && left > 0) at.next_unit(p);
  }
};

// Query row r of unit u: which token and head it is.
__device__ __forceinline__ int row_token(const PagedParams& p, int row) { return row / p.group; }
__device__ __forceinline__ int row_head(const PagedParams& p, int hkv, int row) { return hkv * p.group + row % p.group; }

// The tensor-core kernel (paged_mma.cu).
bool paged_mma_supported(const lh_memref_t* k, const lh_memref_t* v);
int paged_mma_unit_rows(int64_t rows, int D);
int paged_mma_stretches(const lh_ctx* ctx, int64_t rows, int D);
int paged_mma_launch(lh_ctx* ctx, const PagedParams& p, int dtype, int stretches);

}  // namespace lh
