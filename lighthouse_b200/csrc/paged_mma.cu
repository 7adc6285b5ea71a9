// Attention of new tokens over a paged cache of 16-bit rows (16-byte aligned), the kernel that
// serving runs. Per key and kv head it reads 4 D bytes and computes 4 D flop per query row, so
// with the handful of rows that share a kv head it is bound by the cache's bytes from HBM: at
// 6.5 TB/s one SM gets a key of D = 128 every 21 clocks, and everything else only has to fit
// under that. mma.sync does: the products of 16 keys are 16 instructions for up to eight rows
// (tcgen05's 128-row tiles would be filled to a sixteenth, and its operands would have to be
// laid out by one more pass through shared memory for no byte less from HBM).
//
// Both products are taken transposed, S^T = K Q^T and O^T += V^T P^T, so that the long sides (16
// keys, then 16 head dimensions) fill the instruction's m16 and the query rows its n8: eight rows
// cost half of what they would as a half-empty m16, accumulators included. S^T leaves the
// first product with keys along the rows; movmatrix turns its 8 x 8 blocks into the second
// product's operand in registers.
//
// Each warp runs by itself, on its own stretch of tiles: its first lane has the TMA bring 16 keys at a
// time into a ring of the warp's own (one box per 64 dimensions, 128-byte swizzle), and the warp keeps
// its own online softmax, so nothing in the kernel after its first microsecond waits for another
// warp. (With cp.async in its place the addresses of 32 copies per lane and tile were half of all
// instructions, and the kernel was bound by their issue.) Tiles that lie across pages, and pools
// that no tensor map describes, are fetched with cp.async, row by row. At the end of a unit the
// results are turned to rows in the stage just used, while the ring is being filled for the next.
//
// 64 sequences of 133 to 8192 keys (32 heads on 8 of 128, bf16, 1.1 GB) take 187 us in all, 5.9 TB/s or 0.90
// of what a copy reaches; one of 131071 keys 100 us (5.4 TB/s). Shorter calls are bound by what comes
// once: finding the stretches (4000 clocks), a warp's first pages, Q and tiles (5000), a unit's end
// (2000 to 4000) and the join (5 to 10 us): 250 sequences of up to 1024 keys of 12 f16 heads of 64 take 71 us
// (51 for the bytes), 16 of up to 4001 with four new tokens 51 to 56 (21), one of 129 12.3.
#include <type_traits>

#include "paged.cuh"

namespace lh {
namespace {

constexpr int THREADS = 128;
constexpr int SUB = TILE;

// Stages of a warp's ring and CTAs of an SM. A tile takes a warp about 1500 clocks from ldmatrix to the
// next fetch, most of them latency, and its loads are there before it asks for them: more warps
// are worth more than deeper rings, as far as the accumulators leave registers for them.
template <int DP, int NT>
struct Shape {
  static constexpr int stage_bytes = 2 * SUB * DP * 2;  // K and V rows of 16 keys
  static constexpr int ctas_per_sm = DP == 256 ? 1 : NT == 1 ? 3 : 2;
  static constexpr int stages = DP == 64 ? (NT == 1 ? 4 : 6) : DP == 128 ? (NT == 1 ? 2 : 3) : 3;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ float bits_to_f32(uint32_t bits16) {
  if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(static_cast<unsigned short>(bits16)));
  else return __uint_as_float(bits16 << 16);
}

// Where 16-byte chunk `chunk` of row `row` of K or V lies in its half of a stage: blocks of 16 rows x 64
// dimensions, chunks swizzled by the row, as the TMA writes them.
__device__ __forceinline__ uint32_t place_of(int row, int chunk) { return (chunk >> 3) * (SUB * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); }

// The side of a warp that fetches. It knows the next tile and looks pages up ahead of their use: with
// the TMA, where a tile lies within one page, those of 32 tiles at once, one per lane; else those
// of the next tile's 16 keys.
template <typename T, int DP, bool TMA>
struct Producer {
  TileCursor at;
  int64_t left;  // tiles still to fetch
  int page_id, first;  // looked up; the tile that lane 0's page is of
  int hkv;

  __device__ __forceinline__ void begin(const PagedParams& p, const TileCursor& from, int64_t n) {
    at = from;
    left = n;
    enter_unit(p);
  }
  __device__ __forceinline__ void enter_unit(const PagedParams& p) {
    hkv = at.u / p.row_groups;
    look_up(p);
  }
  __device__ __forceinline__ void look_up(const PagedParams& p) {
    const int lane = threadIdx.x & 31;
    first = at.t;
    const int64_t j = TMA ? (static_cast<int64_t>(at.t) + lane) * TILE : at.t * TILE + (lane & 15);
    page_id = j < at.len ? p.table[at.b * p.stb + page_of(p, static_cast<int>(j)) * p.stp] : -1;
  }
  // Starts the copies of the next tile into a stage; returns which of its keys exist. With the TMA they
  // complete on `full`, without on the warp's cp.async group.
  __device__ __forceinline__ uint32_t fetch(const PagedParams& p, const CUtensorMap* tm_k, const CUtensorMap* tm_v, char* stage, uint64_t* full) {
    const int lane = threadIdx.x & 31;
    const int key0 = at.t * TILE;
    constexpr int V_OFF = SUB * DP * 2;
    uint32_t mask;
    if constexpr (TMA) {
      const int id = __shfl_sync(0xffffffffu, page_id, at.t - first);
      const int n = at.len - key0;
      const bool inside = id >= 0 && id < p.num_pages;
      mask = !inside ? 0u : n >= SUB ? 0xffffu : (1u << n) - 1u;
      if (lane == 0) {
        if (inside) {
          const int slot = key0 - page_of(p, key0) * p.page;
          mbar_arrive_expect_tx(full, 2 * V_OFF);
#pragma unroll
          for (int c = 0; c < DP / 64; ++c) {
            tma_load_4d(stage + c * (SUB * 128), tm_k, full, c * 64, slot, hkv, id);
            tma_load_4d(stage + V_OFF + c * (SUB * 128), tm_v, full, c * 64, slot, hkv, id);
          }
        } else {
          report_bad_index(p.dev_status);
        }
      }
    } else {
      constexpr int CHUNKS = DP / 8;             // 16-byte chunks of a row
      constexpr int ROWS_AT_ONCE = 32 / CHUNKS;  // rows that one cp.async per lane covers
      const T* const K = static_cast<const T*>(p.k);
      const T* const V = static_cast<const T*>(p.v);
      const uint32_t to = smem_u32(stage);
      const int chunk = lane % CHUNKS, row_in = lane / CHUNKS;
      const bool chunk_there = chunk * 8 < p.D;
      const int j = key0 + (lane & 15);
      const bool live = j < at.len, inside = page_id >= 0 && page_id < p.num_pages;
      if (live && !inside) report_bad_index(p.dev_status);
      mask = __ballot_sync(0xffffffffu, live && inside) & 0xffffu;
      const int slot = j - page_of(p, j) * p.page;
      const int64_t ko = live && inside ? page_id * p.skp + slot * p.sks + hkv * p.skh : 0;
      const int64_t vo = live && inside ? page_id * p.svp + slot * p.svs + hkv * p.svh : 0;
      if (mask) {
#pragma unroll
        for (int i = 0; i < SUB / ROWS_AT_ONCE; ++i) {
          const int row = i * ROWS_AT_ONCE + row_in;
          const int64_t kr = __shfl_sync(0xffffffffu, ko, row), vr = __shfl_sync(0xffffffffu, vo, row);
          const bool get = chunk_there && (mask >> row & 1);
          const uint32_t dst = to + place_of(row, chunk);
          cp_async16(dst, get ? K + kr + chunk * 8 : K, get ? 16 : 0);
          cp_async16(dst + V_OFF, get ? V + vr + chunk * 8 : V, get ? 16 : 0);
        }
      }
    }
    --left;
    if (++at.t == at.tiles) {
      if (left > 0) {
        at.next_unit(p);
        enter_unit(p);
      }
    } else if (!TMA || at.t - first == 32) {
      look_up(p);
    }
    return mask;
  }
};

template <typename T, int DP, int NT, bool TMA>
__global__ void __launch_bounds__(THREADS, Shape<DP, NT>::ctas_per_sm)
paged_mma_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedParams p) {
  constexpr int STAGES = Shape<DP, NT>::stages, STAGE_BYTES = Shape<DP, NT>::stage_bytes, V_OFF = STAGE_BYTES / 2;
  constexpr int KSTEPS = DP / 16;
  extern __shared__ char smem_raw[];
  __shared__ uint64_t full[4][STAGES];
  __shared__ int gave_up;
  __shared__ uint32_t there[4][STAGES];  // which of a stage's 16 keys exist
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  grid_dependency_trigger();
  if (TMA && threadIdx.x == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    for (int w = 0; w < 4; ++w)
      for (int s = 0; s < STAGES; ++s) mbar_init(&full[w][s], 1);
    gave_up = 0;
    fence_barrier_init();
  }
  TileCursor at;
  int64_t left = find_stretch<THREADS>(p, at);
  if (left == 0) return;  // (its barriers follow the mbarriers' set-up)

  char* const ring = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u) + warp * STAGES * STAGE_BYTES;
  Producer<T, DP, TMA> producer;
  producer.begin(p, at, left);
  auto fetch = [&](int stage) {
    if (producer.left > 0) {
      const uint32_t mask = producer.fetch(p, &tm_k, &tm_v, ring + stage * STAGE_BYTES, &full[warp][stage]);
      if (lane == 0) there[warp][stage] = mask;
    }
    if (!TMA) cp_async_commit();
  };
  uint32_t parity = 0;  // of the next wait on each stage
  auto wait_for = [&](int stage) {
    const bool ok = mbar_wait(&full[warp][stage], parity >> stage & 1, &gave_up, p.dev_status, DEV_TIMEOUT_PAGED);
    parity ^= 1u << stage;
    return __all_sync(0xffffffffu, ok) != 0;
  };

  // ---- a unit: lane r knows query row r of it, the fragments of Q are loaded
  uint32_t qf[NT][KSTEPS][2];
  int64_t o_row;          // lane r: offset of row r of o
  int nrows, seen[NT][2]; // rows; keys that rows 2 t4 and 2 t4 + 1 of each n tile may see
  int t0;
  auto enter_unit = [&]() {
    const int hkv = at.u / p.row_groups, row0 = (at.u - hkv * p.row_groups) * (NT * 8);
    nrows = min(NT * 8, p.rows - row0);
    t0 = at.t;
    const int token = (row0 + lane) / p.group, head = hkv * p.group + (row0 + lane) - token * p.group;
    o_row = at.b * p.sob + head * p.soh + token * p.sos;
    const int64_t q_row = at.b * p.sqb + head * p.sqh + token * p.sqs;
    const int sees = at.len - p.Sq + 1 + token;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      seen[n][0] = __shfl_sync(0xffffffffu, sees, n * 8 + t4 * 2);
      seen[n][1] = __shfl_sync(0xffffffffu, sees, n * 8 + t4 * 2 + 1);
      const bool is = n * 8 + g < nrows;
      const int64_t off = __shfl_sync(0xffffffffu, q_row, n * 8 + g);
      const unsigned short* const q = static_cast<const unsigned short*>(p.q) + (is ? off : 0) + t4 * 2;
      if (p.q_pairs) {
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) qf[n][k][i] = is && k * 16 + i * 8 + t4 * 2 < p.D ? *reinterpret_cast<const uint32_t*>(q + k * 16 + i * 8) : 0u;
      } else {
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const bool in = is && k * 16 + i * 8 + t4 * 2 < p.D;  // D is a multiple of eight
            qf[n][k][i] = in ? q[k * 16 + i * 8] | static_cast<uint32_t>(q[k * 16 + i * 8 + 1]) << 16 : 0u;
          }
      }
    }
  };
  enter_unit();
#pragma unroll
  for (int s = 0; s < STAGES; ++s) fetch(s);

  // ldmatrix addresses inside a stage: lane l gives row (l & 7) of matrix l / 8
  const int mi = lane >> 3, r8 = lane & 7;
  const int krow = (mi & 1) * 8 + r8, kchunk = mi >> 1;  // K: matrices (keys lo, k lo), (keys hi, k lo), (keys lo, k hi), (keys hi, k hi)
  const int vrow = (mi >> 1) * 8 + r8, vchunk = mi & 1;  // V, transposed: (dims lo, keys lo), (dims hi, keys lo), (dims lo, keys hi), (dims hi, keys hi)
  float acc[NT][KSTEPS][4];
  float m[NT][2], l[NT][2];  // query rows 2 t4 and 2 t4 + 1 of each n tile
  auto clear = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][k][i] = 0.f;
    }
  };
  clear();
  int stage = 0;
  for (; left > 0; --left) {
    if (!TMA) cp_async_wait<STAGES - 1>();
    __syncwarp();
    const uint32_t mask = there[warp][stage];
    char* const here = ring + stage * STAGE_BYTES;
    bool wrote = false;  // with plain stores, into a stage that the TMA writes next
    if (mask) {
      const uint32_t base = smem_u32(here);
      const int key0 = at.t * TILE;
      if constexpr (TMA) {
        if (!wait_for(stage)) {  // the copies never came: leave, but let those of the other stages come in
          for (int s = 1; s < STAGES; ++s) {
            const int other = (stage + s) % STAGES;
            int late = 0;
            if (left > s && there[warp][other]) mbar_wait_limit(&full[warp][other], parity >> other & 1, &late, nullptr, 0, LH_WAIT_TIMEOUT_NS);
          }
          return;
        }
        if (mask != 0xffffu) {  // rows behind the last key hold anything: of V, zeros
          wrote = true;
          for (int i = lane; i < SUB * (DP / 8); i += 32) {
            const int row = i / (DP / 8), chunk = i % (DP / 8);
            if (!(mask >> row & 1)) *reinterpret_cast<uint4*>(here + V_OFF + place_of(row, chunk)) = make_uint4(0u, 0u, 0u, 0u);
          }
          __syncwarp();
        }
      }
      float s[NT][4], s2[NT][4];  // even and odd steps: two chains of half the length
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = s2[n][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        uint32_t a[4];
        ldmatrix4(a, base + place_of(krow, k * 2 + kchunk));
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<T>(k & 1 ? s2[n] : s[n], a, qf[n][k][0], qf[n][k][1]);
      }
      const bool some_masked = key0 + SUB > at.len - p.Sq + 1;  // some row does not see some of these keys (or they do not exist)
      const bool whole = mask == 0xffffu && !some_masked;
      bool grows = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][i] = (s[n][i] + s2[n][i]) * p.scale_log2;
          if (!whole) {
            const int key = g + (i >> 1) * 8;
            if (!(mask >> key & 1) || key0 + key >= seen[n][i & 1]) s[n][i] = -INFINITY;
          }
        }
        grows |= fmaxf(s[n][0], s[n][2]) > m[n][0] || fmaxf(s[n][1], s[n][3]) > m[n][1];
      }
      // the running maximum is only brought up to date when some key passes it
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = fmaxf(s[n][i], s[n][i + 2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            top = fmaxf(top, m[n][i]);
            const float alpha = top == -INFINITY ? 1.f : ex2(m[n][i] - top);
            m[n][i] = top;
            l[n][i] *= alpha;
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) {
              acc[n][k][i] *= alpha;
              acc[n][k][i + 2] *= alpha;
            }
          }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float top = m[n][i & 1];
          s[n][i] = ex2(s[n][i] - (top == -INFINITY ? 0.f : top));
        }
        l[n][0] += s[n][0] + s[n][2];
        l[n][1] += s[n][1] + s[n][3];
        pf[n][0] = pack2<T>(s[n][0], s[n][1]);
        pf[n][1] = pack2<T>(s[n][2], s[n][3]);
      }
      if (some_masked && p.Sq > 1) {
        // A weight of zero does not silence a NaN or an infinity in V in the product below. Keys that only
        // the later tokens see are taken out of it when their V is not finite, and added by hand
        // to the rows that do see them.
        bool odd = false;
        for (int r = max(0, at.len - p.Sq + 1 - key0); r < SUB && (mask >> r & 1); ++r)
          for (int c = lane; c < DP; c += 32) {
            const float v = bits_to_f32<T>(*reinterpret_cast<const unsigned short*>(here + V_OFF + place_of(r, c >> 3) + (c & 7) * 2));
            odd |= !(fabsf(v) < INFINITY);
          }
        if (__any_sync(0xffffffffu, odd)) {
          wrote = true;
          for (int r = max(0, at.len - p.Sq + 1 - key0); r < SUB; ++r) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint32_t two = __shfl_sync(0xffffffffu, r < 8 ? pf[n][0] : pf[n][1], (r & 7) * 4 + t4);
              const float p0 = bits_to_f32<T>(two & 0xffffu), p1 = bits_to_f32<T>(two >> 16);
#pragma unroll
              for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const float v = bits_to_f32<T>(*reinterpret_cast<const unsigned short*>(here + V_OFF + place_of(r, k * 2 + i) + g * 2));
                  if (p0 != 0.f) acc[n][k][i * 2] = fmaf(p0, v, acc[n][k][i * 2]);
                  if (p1 != 0.f) acc[n][k][i * 2 + 1] = fmaf(p1, v, acc[n][k][i * 2 + 1]);
                }
            }
            __syncwarp();
            for (int c = lane; c < DP / 8; c += 32) *reinterpret_cast<uint4*>(here + V_OFF + place_of(r, c)) = make_uint4(0u, 0u, 0u, 0u);
          }
          __syncwarp();
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        pf[n][0] = movmatrix_trans(pf[n][0]);
        pf[n][1] = movmatrix_trans(pf[n][1]);
      }
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        uint32_t a[4];
        ldmatrix4_trans(a, base + V_OFF + place_of(vrow, k * 2 + vchunk));
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<T>(acc[n][k], a, pf[n][0], pf[n][1]);
      }
    }
    __syncwarp();
    if (++at.t == at.tiles || left == 1) {
      // ---- the warp leaves the unit. The stage just used takes two n tiles of results as rows of f32;
      // dimensions are swizzled by the row so that neither side meets in a bank. The next unit's
      // Q is on its way meanwhile.
      float* const buf = reinterpret_cast<float*>(here);
      wrote = true;
      const int64_t slot = partial_slot<THREADS>(t0, at.t, at.tiles);
      const int64_t rows_at = slot < 0 ? o_row : (slot * p.part_rows + lane) * p.Dp;
      const int n_done = nrows;
      if (left > 1) {
        at.next_unit(p);
        enter_unit();
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], d);
      if (slot >= 0 && g == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (n * 8 + t4 * 2 + i < n_done) p.ml[slot * p.part_rows + n * 8 + t4 * 2 + i] = make_float2(m[n][i], l[n][i]);
      }
#pragma unroll
      for (int n0 = 0; n0 < NT; n0 += 2) {
#pragma unroll
        for (int n = n0; n < NT && n < n0 + 2; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            // a row that sees no key has no weight: zeros
            const float inv = slot >= 0 ? 1.f : l[n][i] == 0.f ? 0.f : 1.f / l[n][i];
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
              for (int e = 0; e < 2; ++e) buf[((n - n0) * 8 + t4 * 2 + i) * DP + ((k * 16 + e * 8 + g) ^ (t4 << 3))] = acc[n][k][e * 2 + i] * inv;
          }
        __syncwarp();
#pragma unroll 4
        for (int q = 0; q < 16; ++q) {
          const int r = n0 * 8 + q;
          if (r >= n_done || (NT == 1 && q >= 8)) break;
          const int64_t to = __shfl_sync(0xffffffffu, rows_at, r);
#pragma unroll
          for (int d0 = 0; d0 < DP; d0 += 128) {
            const int d = d0 + lane * 4;
            if (d >= DP) break;
            const float4 v = *reinterpret_cast<const float4*>(buf + q * DP + (d ^ ((q >> 1 & 3) << 3)));
            if (slot < 0) store_o4(p, to, d, v);
            else if (d < p.Dp) *reinterpret_cast<float4*>(p.part + to + d) = v;
          }
        }
        __syncwarp();
      }
      clear();
    }
    if (TMA && wrote) {
      fence_proxy_async_smem();
      __syncwarp();
    }
    fetch(stage);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
}

// Query rows of a unit: eight, sixteen or thirty-two, whichever takes the rows of a kv head in
// the fewest passes over its keys (32 x 256 accumulators would not fit the registers).
int n_tiles_for(int rows, int D) {
  const int most = D > 128 ? 2 : 4;
  return rows <= 8 ? 1 : rows <= 16 || most == 2 ? 2 : 4;
}

// A pool as a tensor (dimension, row of a page, head, page) for the TMA; false where that cannot be: tiles
// across pages, an empty pool, strides that repeat elements.
bool encode_pool(lh_ctx* ctx, CUtensorMap* map, int dtype, const void* base, const PagedParams& p, int64_t slot, int64_t head, int64_t page) {
  if (p.page % TILE || p.num_pages < 1) return false;
  const uint64_t dims[4] = {static_cast<uint64_t>(p.D), static_cast<uint64_t>(p.page), static_cast<uint64_t>(p.Hkv), static_cast<uint64_t>(p.num_pages)};
  uint64_t strides[3];
  const int64_t elements[3] = {slot, head, page};
  for (int i = 0; i < 3; ++i) {
    if (dims[i + 1] > 1 && (elements[i] <= 0 || elements[i] >= int64_t(1) << 38)) return false;
    strides[i] = dims[i + 1] > 1 ? static_cast<uint64_t>(elements[i]) * 2 : 16;
  }
  const uint32_t box[4] = {64, TILE, 1, 1};
  return encode_tensor_map(ctx, map, dtype, 4, const_cast<void*>(base), dims, strides, box, 1) == LH_OK;
}

template <typename T, int DP, int NT>
int launch(lh_ctx* ctx, const PagedParams& p, int ctas) {
  constexpr int smem = THREADS / 32 * Shape<DP, NT>::stages * Shape<DP, NT>::stage_bytes + 1024;  // the swizzle wants 1024-byte boundaries
  const int dtype = std::is_same<T, __half>::value ? LH_F16 : LH_BF16;
  CUtensorMap k, v;
  memset(&k, 0, sizeof(k));
  memset(&v, 0, sizeof(v));
  const bool tma = encode_pool(ctx, &k, dtype, p.k, p, p.sks, p.skh, p.skp) && encode_pool(ctx, &v, dtype, p.v, p, p.svs, p.svh, p.svp);
  auto* kernel = tma ? paged_mma_kernel<T, DP, NT, true> : paged_mma_kernel<T, DP, NT, false>;
  LH_CUDA_CHECK(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kernel<<<static_cast<unsigned>(ctas), THREADS, smem, ctx->stream>>>(k, v, p);
  LH_CHECK_LAUNCH(ctx, "paged_mma_kernel");
  return LH_OK;
}
template <typename T>
int launch_type(lh_ctx* ctx, const PagedParams& p, int ctas) {
  const int nt = p.unit_rows / 8;
  if (p.D <= 64) return nt == 1 ? launch<T, 64, 1>(ctx, p, ctas) : nt == 2 ? launch<T, 64, 2>(ctx, p, ctas) : launch<T, 64, 4>(ctx, p, ctas);
  if (p.D <= 128) return nt == 1 ? launch<T, 128, 1>(ctx, p, ctas) : nt == 2 ? launch<T, 128, 2>(ctx, p, ctas) : launch<T, 128, 4>(ctx, p, ctas);
  return nt == 1 ? launch<T, 256, 1>(ctx, p, ctas) : launch<T, 256, 2>(ctx, p, ctas);
}

}  // namespace

int paged_mma_unit_rows(int64_t rows, int D) { return 8 * n_tiles_for(rows > 64 ? 64 : static_cast<int>(rows), D); }
int paged_mma_stretches(const lh_ctx* ctx, int64_t rows, int D) {
  const bool one = paged_mma_unit_rows(rows, D) == 8;
  const int ctas = D > 128 ? Shape<256, 1>::ctas_per_sm : one ? Shape<128, 1>::ctas_per_sm : Shape<128, 2>::ctas_per_sm;
  static_assert(Shape<64, 1>::ctas_per_sm == Shape<128, 1>::ctas_per_sm && Shape<64, 2>::ctas_per_sm == Shape<128, 2>::ctas_per_sm && Shape<256, 1>::ctas_per_sm == Shape<256, 2>::ctas_per_sm && Shape<128, 2>::ctas_per_sm == Shape<128, 4>::ctas_per_sm, "one rule for all");
  return THREADS / 32 * ctx->sm_count * ctas;
}

bool paged_mma_supported(const lh_memref_t* k, const lh_memref_t* v) {
  if ((k->dtype != LH_BF16 && k->dtype != LH_F16) || k->shape[3] % 8) return false;
  for (const lh_memref_t* m : {k, v}) {
    if (reinterpret_cast<uintptr_t>(data_ptr(m)) % 16) return false;
    for (int i = 0; i < 3; ++i)
      if (m->shape[i] > 1 && m->strides[i] % 8) return false;
  }
  return true;
}

int paged_mma_launch(lh_ctx* ctx, const PagedParams& p, int dtype, int stretches) {
  const int ctas = stretches / (THREADS / 32);
  return dtype == LH_BF16 ? launch_type<__nv_bfloat16>(ctx, p, ctas) : launch_type<__half>(ctx, p, ctas);
}

}  // namespace lh
