// The paged key-value cache: writing new rows into it (rotary embedding fused in) and
// attending over it. Entry points lh_b200_paged_append, lh_b200_paged_attention.
#include <type_traits>

#include "paged.cuh"

namespace lh {
namespace {

// ------------------------------------------------------------------- append
// For token t: q <- rot(q, pos[t]) in place, page rows of slot[t] <- rot(k, pos[t]) and v.
// A pure copy: bound by the bytes of q (twice), k, v and their cache rows, and for a few
// tokens by latency. One CTA (or several, below) per token: the D/2 angles are computed once
// into shared memory and used by every head.
struct AppendParams {
  void* q; const void* k; const void* v; void* kp; void* vp;
  const void* slots; const void* pos;
  int64_t sqt, sqh, skt, skh, svt, svh;
  int64_t kpp, kps, kph, vpp, vps, vph;
  int64_t sslot, spos;
  int64_t num_slots;
  int Hq, Hkv, D, page;
  int q_dtype, c_dtype;
  int slots64, pos64, rotate;
  double log2_theta;
  int* dev_status;
};

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int wide) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// pos * theta^(-2i/D) is formed and reduced in f64: at position 10^6 an f32 product is already
// off by 0.03 rad. What is left lies in [-pi, pi], where f32 sine and cosine are exact to 1e-7.
__device__ __forceinline__ float2 rope_angle(double log2_theta, int i, int dim, int64_t pos) {
  const double freq = exp2(-static_cast<double>(2 * i) / dim * log2_theta);
  const double ang = static_cast<double>(pos) * freq;
  const double two_pi = 6.283185307179586476925;
  const float r = static_cast<float>(ang - two_pi * rint(ang / two_pi));
  float s, c;
  sincosf(r, &s, &c);
  return make_float2(c, s);
}

constexpr int APPEND_THREADS = 256;
constexpr int APPEND_MAX_PAIRS = 256;  // head sizes up to 512

template <typename T>
struct Vec8;
template <>
struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0]; b = reinterpret_cast<const float4*>(p)[1]; }
  __device__ __forceinline__ void store(float* p) const { reinterpret_cast<float4*>(p)[0] = a; reinterpret_cast<float4*>(p)[1] = b; }
  __device__ __forceinline__ void get(float (&f)[8]) const { f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w; }
  __device__ __forceinline__ void set(const float (&f)[8]) { a = make_float4(f[0], f[1], f[2], f[3]); b = make_float4(f[4], f[5], f[6], f[7]); }
};
template <>
struct Vec8<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = a; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&a);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 x = __bfloat1622float2(h[i]); f[2 * i] = x.x; f[2 * i + 1] = x.y; }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&a);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  }
};
template <>
struct Vec8<__half> {
  uint4 a;
  __device__ __forceinline__ void load(const __half* p) { a = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(__half* p) const { *reinterpret_cast<uint4*>(p) = a; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const __half2* h = reinterpret_cast<const __half2*>(&a);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 x = __half22float2(h[i]); f[2 * i] = x.x; f[2 * i + 1] = x.y; }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    __half2* h = reinterpret_cast<__half2*>(&a);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  }
};

// Rows of 16-byte aligned groups of eight elements. Values are rotated in f32 and rounded once
// to the type they are stored in.
template <typename TQ, typename TC>
__global__ void __launch_bounds__(APPEND_THREADS) append_vec_kernel(const AppendParams p) {
  __shared__ float2 angle[APPEND_MAX_PAIRS];
  const int64_t t = blockIdx.x;
  const int64_t slot = load_index(p.slots, t * p.sslot, p.slots64);
  if (p.rotate) {
    const int64_t pos = load_index(p.pos, t * p.spos, p.pos64);
    for (int i = threadIdx.x; i < p.D / 2; i += APPEND_THREADS) angle[i] = rope_angle(p.log2_theta, i, p.D, pos);
    __syncthreads();
  }
  const bool bad = slot >= p.num_slots;
  if (bad && threadIdx.x == 0 && blockIdx.y == 0) report_bad_index(p.dev_status);
  const bool keep = slot >= 0 && !bad;
  const int64_t pg = keep ? slot / p.page : 0, at = keep ? slot % p.page : 0;
  const int cols = p.D / 8;
  const int units = (p.Hq + 2 * p.Hkv) * cols;
  for (int u = blockIdx.y * APPEND_THREADS + threadIdx.x; u < units; u += gridDim.y * APPEND_THREADS) {
    const int head = u / cols, col = u - head * cols;
    float f[8];
    Vec8<TQ> in;
    if (head < p.Hq + p.Hkv) {
      const bool is_q = head < p.Hq;
      if (is_q && !p.rotate) continue;
      if (!is_q && !keep) continue;
      const int h = is_q ? head : head - p.Hq;
      const TQ* src = is_q ? static_cast<const TQ*>(p.q) + t * p.sqt + h * p.sqh + col * 8 : static_cast<const TQ*>(p.k) + t * p.skt + h * p.skh + col * 8;
      in.load(src);
      in.get(f);
      if (p.rotate) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 cs = angle[col * 4 + i];
          const float x = f[2 * i], y = f[2 * i + 1];
          f[2 * i] = x * cs.x - y * cs.y;
          f[2 * i + 1] = x * cs.y + y * cs.x;
        }
      }
      if (is_q) {
        in.set(f);
        in.store(static_cast<TQ*>(p.q) + t * p.sqt + h * p.sqh + col * 8);
      } else {
        Vec8<TC> out;
        out.set(f);
        out.store(static_cast<TC*>(p.kp) + pg * p.kpp + at * p.kps + h * p.kph + col * 8);
      }
    } else if (keep) {
      const int h = head - p.Hq - p.Hkv;
      in.load(static_cast<const TQ*>(p.v) + t * p.svt + h * p.svh + col * 8);
      TC* dst = static_cast<TC*>(p.vp) + pg * p.vpp + at * p.vps + h * p.vph + col * 8;
      if constexpr (std::is_same<TQ, TC>::value) {
        in.store(dst);
      } else {
        Vec8<TC> out;
        in.get(f);
        out.set(f);
        out.store(dst);
      }
    }
  }
}

// Any alignment, stride and (without rotation) odd head size: one pair of elements per thread.
__global__ void __launch_bounds__(APPEND_THREADS) append_generic_kernel(const AppendParams p) {
  __shared__ float2 angle[APPEND_MAX_PAIRS];
  const int64_t t = blockIdx.x;
  const int64_t slot = load_index(p.slots, t * p.sslot, p.slots64);
  if (p.rotate) {
    const int64_t pos = load_index(p.pos, t * p.spos, p.pos64);
    for (int i = threadIdx.x; i < p.D / 2; i += APPEND_THREADS) angle[i] = rope_angle(p.log2_theta, i, p.D, pos);
    __syncthreads();
  }
  const bool bad = slot >= p.num_slots;
  if (bad && threadIdx.x == 0 && blockIdx.y == 0) report_bad_index(p.dev_status);
  const bool keep = slot >= 0 && !bad;
  const int64_t pg = keep ? slot / p.page : 0, at = keep ? slot % p.page : 0;
  const int cols = (p.D + 1) / 2;
  const int units = (p.Hq + 2 * p.Hkv) * cols;
  for (int u = blockIdx.y * APPEND_THREADS + threadIdx.x; u < units; u += gridDim.y * APPEND_THREADS) {
    const int head = u / cols, d = 2 * (u - head * cols);
    const bool two = d + 1 < p.D;
    if (head < p.Hq + p.Hkv) {
      const bool is_q = head < p.Hq;
      if (is_q ? !p.rotate : !keep) continue;
      const int h = is_q ? head : head - p.Hq;
      const void* src = is_q ? p.q : p.k;
      const int64_t off = (is_q ? t * p.sqt + h * p.sqh : t * p.skt + h * p.skh) + d;
      float x = load_as_f32(src, p.q_dtype, off), y = two ? load_as_f32(src, p.q_dtype, off + 1) : 0.f;
      if (p.rotate) {
        const float2 cs = angle[d / 2];
        const float x0 = x;
        x = x0 * cs.x - y * cs.y;
        y = x0 * cs.y + y * cs.x;
      }
      void* dst = is_q ? p.q : p.kp;
      const int dt = is_q ? p.q_dtype : p.c_dtype;
      const int64_t to = is_q ? off : pg * p.kpp + at * p.kps + h * p.kph + d;
      store_from_f32(dst, dt, to, x);
      if (two) store_from_f32(dst, dt, to + 1, y);
    } else if (keep) {
      const int h = head - p.Hq - p.Hkv;
      const int64_t off = t * p.svt + h * p.svh + d, to = pg * p.vpp + at * p.vps + h * p.vph + d;
      store_from_f32(p.vp, p.c_dtype, to, load_as_f32(p.v, p.q_dtype, off));
      if (two) store_from_f32(p.vp, p.c_dtype, to + 1, load_as_f32(p.v, p.q_dtype, off + 1));
    }
  }
}

typedef void (*AppendKernel)(const AppendParams);
AppendKernel append_vec_for(int q_dtype, int c_dtype) {
#define LH_APPEND_ROW(TQ)                                             \
  switch (c_dtype) {                                                  \
    case LH_F32: return append_vec_kernel<TQ, float>;                 \
    case LH_BF16: return append_vec_kernel<TQ, __nv_bfloat16>;        \
    default: return append_vec_kernel<TQ, __half>;                    \
  }
  switch (q_dtype) {
    case LH_F32: LH_APPEND_ROW(float)
    case LH_BF16: LH_APPEND_ROW(__nv_bfloat16)
    default: LH_APPEND_ROW(__half)
  }
#undef LH_APPEND_ROW
}

// ---------------------------------------------------------------- attention
// The general kernel: f32 caches, and 16-bit ones whose rows are not 16-byte aligned. Scores
// with one key per lane, P V with four head dimensions per lane, both on FFMA; K and V come
// straight from global memory (a K row is read 16 bytes at a time by its lane, the rest of
// the sector from L1). Each warp keeps an online softmax of its own over its 32 keys of every
// tile; the four are joined when the CTA leaves a unit.
constexpr int SIMT_THREADS = 128;
constexpr int SIMT_ROWS = 8;
constexpr int SIMT_TILE = 128;
constexpr int SIMT_CTAS_PER_SM = 4;

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}

// Four elements from `d` on; elements at D and beyond read as zero.
template <typename T, bool VEC>
__device__ __forceinline__ float4 load4(const T* row, int d, int D) {
  if constexpr (VEC) {  // D and every offset are multiples of four elements
    if (d >= D) return make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (std::is_same<T, float>::value) {
      return *reinterpret_cast<const float4*>(row + d);
    } else {
      const uint2 raw = *reinterpret_cast<const uint2*>(row + d);
      const T* e = reinterpret_cast<const T*>(&raw);
      return make_float4(to_f32(e[0]), to_f32(e[1]), to_f32(e[2]), to_f32(e[3]));
    }
  } else {
    return make_float4(d < D ? to_f32(row[d]) : 0.f, d + 1 < D ? to_f32(row[d + 1]) : 0.f, d + 2 < D ? to_f32(row[d + 2]) : 0.f, d + 3 < D ? to_f32(row[d + 3]) : 0.f);
  }
}

template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(SIMT_THREADS) paged_simt_kernel(const PagedParams p) {
  constexpr int DMAX = NV * 128;
  __shared__ __align__(16) float qs[SIMT_ROWS][DMAX];  // read four at a time
  __shared__ __align__(16) float obuf[SIMT_ROWS][DMAX];
  __shared__ float ps[4][SIMT_ROWS][32];
  __shared__ float wm[4][SIMT_ROWS], wl[4][SIMT_ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dependency_trigger();
  int64_t lo, hi;
  TileCursor at;
  if (!find_stretch<SIMT_THREADS>(p, lo, hi, at)) return;
  const T* K = static_cast<const T*>(p.k);
  const T* V = static_cast<const T*>(p.v);
  while (lo < hi) {
    const int t0 = at.t;
    const int t1 = static_cast<int>(at.tiles - t0 <= hi - lo ? at.tiles : t0 + (hi - lo));
    const int hkv = at.u / p.row_groups, row0 = (at.u % p.row_groups) * SIMT_ROWS;
    const int nrows = min(SIMT_ROWS, p.rows - row0);
    for (int i = tid; i < SIMT_ROWS * DMAX; i += SIMT_THREADS) {
      const int r = i / DMAX, d = i % DMAX;
      float x = 0.f;
      if (r < nrows && d < p.D) {
        const int row = row0 + r;
        x = to_f32(static_cast<const T*>(p.q)[at.b * p.sqb + row_head(p, hkv, row) * p.sqh + row_token(p, row) * p.sqs + d]) * p.scale_log2;
      }
      qs[r][d] = x;
    }
    __syncthreads();
    float m[SIMT_ROWS], l[SIMT_ROWS], acc[SIMT_ROWS][NV * 4];
    int seen[SIMT_ROWS];  // keys that the row may attend to
#pragma unroll
    for (int r = 0; r < SIMT_ROWS; ++r) {
      seen[r] = r < nrows ? at.len - p.Sq + 1 + row_token(p, row0 + r) : 0;
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV * 4; ++i) acc[r][i] = 0.f;
    }
    for (int t = t0; t < t1; ++t) {
      const int first = t * SIMT_TILE + warp * 32;
      if (first >= at.len) break;
      const int j = first + lane;
      int64_t koff = -1, voff = -1;
      if (j < at.len) {
        const int pg = page_of(p, j), slot = j - pg * p.page;
        const int64_t id = p.table[at.b * p.stb + pg * p.stp];
        if (id >= 0 && id < p.num_pages) {
          koff = id * p.skp + slot * p.sks + hkv * p.skh;
          voff = id * p.svp + slot * p.svs + hkv * p.svh;
        } else {
          report_bad_index(p.dev_status);
        }
      }
      const bool live = koff >= 0;
      float s[SIMT_ROWS];
#pragma unroll
      for (int r = 0; r < SIMT_ROWS; ++r) s[r] = 0.f;
      if (live) {
#pragma unroll 4
        for (int d = 0; d < p.D; d += 4) {
          const float4 kv = load4<T, VEC>(K + koff, d, p.D);
#pragma unroll
          for (int r = 0; r < SIMT_ROWS; ++r) {
            const float4 qv = *reinterpret_cast<const float4*>(&qs[r][d]);
            s[r] = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, fmaf(qv.z, kv.z, fmaf(qv.w, kv.w, s[r]))));
          }
        }
      }
      // keys that only the later of several new tokens may see: masked rows must not meet their V
      const bool partial = first + 32 > at.len - p.Sq + 1;
#pragma unroll
      for (int r = 0; r < SIMT_ROWS; ++r) {
        if (!live || j >= seen[r]) s[r] = -INFINITY;
        float top = s[r];
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        top = fmaxf(top, m[r]);
        const float alpha = exp2_safe(m[r], top), e = exp2_safe(s[r], top);
        m[r] = top;
        l[r] = l[r] * alpha + e;
        ps[warp][r][lane] = e;
#pragma unroll
        for (int i = 0; i < NV * 4; ++i) acc[r][i] *= alpha;
      }
      __syncwarp();
#pragma unroll 4
      for (int jj = 0; jj < 32; ++jj) {
        const int64_t off = __shfl_sync(0xffffffffu, voff, jj);
        if (off < 0) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const float4 vv = load4<T, VEC>(V + off, i * 128 + lane * 4, p.D);
#pragma unroll
          for (int r = 0; r < SIMT_ROWS; ++r) {
            const float e = ps[warp][r][jj];
            if (partial && e == 0.f) continue;
            acc[r][i * 4 + 0] = fmaf(e, vv.x, acc[r][i * 4 + 0]);
            acc[r][i * 4 + 1] = fmaf(e, vv.y, acc[r][i * 4 + 1]);
            acc[r][i * 4 + 2] = fmaf(e, vv.z, acc[r][i * 4 + 2]);
            acc[r][i * 4 + 3] = fmaf(e, vv.w, acc[r][i * 4 + 3]);
          }
        }
      }
      __syncwarp();
    }
    // join the four warps
#pragma unroll
    for (int r = 0; r < SIMT_ROWS; ++r) {
#pragma unroll
      for (int d = 16; d; d >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
      if (lane == 0) {
        wm[warp][r] = m[r];
        wl[warp][r] = l[r];
      }
    }
    __syncthreads();
    for (int w = 0; w < 4; ++w) {
      if (w == warp) {
#pragma unroll
        for (int r = 0; r < SIMT_ROWS; ++r) {
          const float M = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r]));
          const float f = exp2_safe(m[r], M);
#pragma unroll
          for (int i = 0; i < NV * 4; ++i) {
            float* o = &obuf[r][(i / 4) * 128 + lane * 4 + (i & 3)];
            // a warp without keys adds nothing (its sums are zeros)
            *o = w == 0 ? acc[r][i] * f : fmaf(acc[r][i], f, *o);
          }
        }
      }
      __syncthreads();
    }
    const int64_t slot = partial_slot(t0, t1, at.tiles);
    for (int i = tid; i < nrows * p.D; i += SIMT_THREADS) {
      const int r = i / p.D, d = i % p.D, row = row0 + r;
      const float M = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r]));
      float L = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) L += wl[w][r] * exp2_safe(wm[w][r], M);
      if (slot < 0) {
        store_from_f32(p.o, p.o_dtype, at.b * p.sob + row_head(p, hkv, row) * p.soh + row_token(p, row) * p.sos + d, L == 0.f ? 0.f : obuf[r][d] / L);
      } else {
        p.part[(slot * p.unit_rows + r) * p.Dp + d] = obuf[r][d];
        if (d == 0) p.ml[slot * p.unit_rows + r] = make_float2(M, L);
      }
    }
    __syncthreads();
    lo += t1 - t0;
    at.t = t1;
    if (lo < hi && at.t == at.tiles) at.next_unit(p);
  }
}

// Joins the units that several CTAs worked on: block i looks at the border between stretch
// i - 1 and stretch i, and if it is the first border inside a unit, adds up that unit's parts
// (8 warps take the parts in turn, a lane holds four head dimensions). The order of the sum is
// fixed by the stretches. It also writes the zeros of sequences that hold no keys. A programmatic
// dependent of the kernel above: it is resident and waiting when that one ends.
constexpr int JOIN_THREADS = 256;
__global__ void __launch_bounds__(JOIN_THREADS) paged_join_kernel(const PagedParams p) {
  __shared__ float red[JOIN_THREADS / 32];
  __shared__ float4 sums[JOIN_THREADS / 32][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dependency_wait();
  if (blockIdx.y == 0) {
    const int64_t per = static_cast<int64_t>(p.Hkv) * p.group * p.Sq * p.D;
    for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
      if (paged_length(p, b)) continue;
      for (int64_t i = tid; i < per; i += JOIN_THREADS) {
        const int d = static_cast<int>(i % p.D);
        const int64_t rest = i / p.D;
        store_from_f32(p.o, p.o_dtype, b * p.sob + (rest / p.Sq) * p.soh + (rest % p.Sq) * p.sos + d, 0.f);
      }
    }
  }
  if (blockIdx.x == 0) return;
  const int4 here = p.first[blockIdx.x];
  if (here.x < 0 || here.z == 0) return;  // no stretch, or one that begins with its unit
  const int64_t total = *p.total;
  const int64_t n = total < gridDim.x ? total : gridDim.x;
  const int64_t lo = stretch_begin(total, n, blockIdx.x);
  const int64_t begin = lo - here.z;
  if (stretch_begin(total, n, blockIdx.x - 1) > begin) return;  // an earlier block has this unit
  const int len = paged_length(p, here.x);
  const int64_t end = begin + paged_tiles(p, len);
  const int64_t c0 = blockIdx.x - 1;
  const int parts = static_cast<int>(stretch_owner(total, n, end - 1) - c0 + 1);
  auto slot_of = [&](int c) { return c == 0 ? 2 * c0 + 1 : 2 * (c0 + c); };
  const int hkv = here.y / p.row_groups, row0 = (here.y % p.row_groups) * p.unit_rows;
  const int nrows = min(p.unit_rows, p.rows - row0);
  for (int r = blockIdx.y; r < nrows; r += gridDim.y) {
    float M = -INFINITY;
    for (int c = tid; c < parts; c += JOIN_THREADS) M = fmaxf(M, p.ml[slot_of(c) * p.unit_rows + r].x);
#pragma unroll
    for (int d = 16; d; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    if (lane == 0) red[warp] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < JOIN_THREADS / 32; ++w) M = fmaxf(M, red[w]);
    const int row = row0 + r;
    const int64_t out = here.x * p.sob + row_head(p, hkv, row) * p.soh + row_token(p, row) * p.sos;
    for (int d0 = 0; d0 < p.Dp; d0 += 128) {
      const int d = d0 + lane * 4;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      float L = 0.f;
      for (int c = warp; c < parts; c += JOIN_THREADS / 32) {
        const int64_t at = slot_of(c) * p.unit_rows + r;
        const float2 ml = p.ml[at];
        const float f = exp2_safe(ml.x, M);
        L = fmaf(ml.y, f, L);
        if (d < p.Dp) {
          const float4 x = *reinterpret_cast<const float4*>(p.part + at * p.Dp + d);
          a.x = fmaf(x.x, f, a.x); a.y = fmaf(x.y, f, a.y); a.z = fmaf(x.z, f, a.z); a.w = fmaf(x.w, f, a.w);
        }
      }
      __syncthreads();
      sums[warp][lane] = a;
      if (lane == 0) red[warp] = L;
      __syncthreads();
      if (warp == 0) {
        L = 0.f;
        a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < JOIN_THREADS / 32; ++w) {
          const float4 x = sums[w][lane];
          a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
          L += red[w];
        }
        // a row that sees no key has no weight at all: zeros
        const float inv = L == 0.f ? 0.f : 1.f / L;
        if (d < p.D) store_from_f32(p.o, p.o_dtype, out + d, a.x * inv);
        if (d + 1 < p.D) store_from_f32(p.o, p.o_dtype, out + d + 1, a.y * inv);
        if (d + 2 < p.D) store_from_f32(p.o, p.o_dtype, out + d + 2, a.z * inv);
        if (d + 3 < p.D) store_from_f32(p.o, p.o_dtype, out + d + 3, a.w * inv);
      }
    }
    __syncthreads();
  }
}

int join_launch(lh_ctx* ctx, const PagedParams& p, int ctas) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(p.rows < p.unit_rows ? p.rows : p.unit_rows));
  cfg.blockDim = dim3(JOIN_THREADS);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LH_CUDA_CHECK(ctx, cudaLaunchKernelEx(&cfg, paged_join_kernel, p));
  LH_CHECK_LAUNCH(ctx, "paged_join_kernel");
  return LH_OK;
}

typedef void (*PagedKernel)(const PagedParams);
template <typename T>
PagedKernel simt_kernel_for(int D, bool vec) {
  if (D <= 128) return vec ? paged_simt_kernel<T, 1, true> : paged_simt_kernel<T, 1, false>;
  return vec ? paged_simt_kernel<T, 2, true> : paged_simt_kernel<T, 2, false>;
}

bool aligned_view(const lh_memref_t* m, int elems) {
  if (reinterpret_cast<uintptr_t>(data_ptr(m)) % (elems * dtype_size(m->dtype))) return false;
  for (int i = 0; i + 1 < m->rank; ++i)
    if (m->shape[i] > 1 && m->strides[i] % elems) return false;
  return true;
}

bool float_type(int dt) { return dt == LH_F32 || dt == LH_BF16 || dt == LH_F16; }

// A view that is written: no element of it may be two elements.
bool overlaps_itself(const lh_memref_t* m) {
  for (int i = 0; i < m->rank; ++i)
    if (m->shape[i] > 1 && m->strides[i] == 0) return true;
  return false;
}

bool sane_extents(const lh_memref_t* m) {
  for (int i = 0; i < m->rank; ++i)
    if (m->shape[i] < 0 || m->shape[i] > 0x7fffffffll) return false;
  return true;
}

struct Workspace {
  size_t first, ml, part, bytes;
};
Workspace workspace_for(int64_t ctas, int unit_rows, int Dp) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  Workspace w;
  w.first = 256;  // the tile count comes first
  w.ml = w.first + up(ctas * sizeof(int4));
  w.part = w.ml + up(2 * ctas * unit_rows * sizeof(float2));
  w.bytes = w.part + up(2 * ctas * static_cast<size_t>(unit_rows) * Dp * sizeof(float));
  return w;
}

int check_attention(lh_ctx* ctx, const lh_memref_t* o, const lh_memref_t* q, const lh_memref_t* k, const lh_memref_t* v, const lh_memref_t* table, const lh_memref_t* lengths) {
  if (!o || !q || !k || !v || !table || !lengths) return set_error(ctx, LH_ERR_INVALID, "paged_attention: o, q, k_pages, v_pages, page_table and lengths are required");
  if (q->rank != 4 || o->rank != 4) return set_error(ctx, LH_ERR_INVALID, "paged_attention: q and o are rank-4 (B, Hq, S, D) views");
  if (k->rank != 4 || v->rank != 4) return set_error(ctx, LH_ERR_INVALID, "paged_attention: k_pages and v_pages are rank-4 (pages, page_size, Hkv, D) views");
  if (table->rank != 2 || lengths->rank != 1) return set_error(ctx, LH_ERR_INVALID, "paged_attention: page_table is (B, columns), lengths is (B)");
  if (!sane_extents(o) || !sane_extents(q) || !sane_extents(k) || !sane_extents(v) || !sane_extents(table) || !sane_extents(lengths))
    return set_error(ctx, LH_ERR_INVALID, "paged_attention: extent out of range");
  for (int i = 0; i < 4; ++i) {
    if (o->shape[i] != q->shape[i]) return set_error(ctx, LH_ERR_INVALID, "paged_attention: o must have q's shape");
    if (v->shape[i] != k->shape[i]) return set_error(ctx, LH_ERR_INVALID, "paged_attention: v_pages must have k_pages's shape");
  }
  if (table->shape[0] != q->shape[0] || lengths->shape[0] != q->shape[0]) return set_error(ctx, LH_ERR_INVALID, "paged_attention: page_table and lengths must have q's batch size");
  if (k->shape[3] != q->shape[3] || q->shape[3] < 1) return set_error(ctx, LH_ERR_INVALID, "paged_attention: head sizes of q and the pages differ, or are zero");
  if (k->shape[2] < 1 || q->shape[1] % k->shape[2]) return set_error(ctx, LH_ERR_INVALID, "paged_attention: %lld query heads are not a multiple of %lld kv heads", (long long)q->shape[1], (long long)k->shape[2]);
  if (k->shape[1] < 1) return set_error(ctx, LH_ERR_INVALID, "paged_attention: page size must be at least 1");
  if (table->dtype != LH_I32 || lengths->dtype != LH_I32) return set_error(ctx, LH_ERR_INVALID, "paged_attention: page_table and lengths are i32");
  if (q->dtype != k->dtype || q->dtype != v->dtype) return set_error(ctx, LH_ERR_INVALID, "paged_attention: q and the pages must have one type");
  if (!float_type(q->dtype) || !float_type(o->dtype)) return set_error(ctx, LH_ERR_UNSUPPORTED, "paged_attention: f32, bf16 or f16 operands");
  if (q->shape[3] > 256) return set_error(ctx, LH_ERR_UNSUPPORTED, "paged_attention: head size %lld is above 256", (long long)q->shape[3]);
  for (const lh_memref_t* m : {o, q, k, v})
    if (m->shape[3] > 1 && m->strides[3] != 1) return set_error(ctx, LH_ERR_UNSUPPORTED, "paged_attention: the head dimension must have unit stride");
  if (overlaps_itself(o)) return set_error(ctx, LH_ERR_INVALID, "paged_attention: o overlaps itself (zero stride)");
  if (table->shape[1] * k->shape[1] > 0x7fffff00ll) return set_error(ctx, LH_ERR_UNSUPPORTED, "paged_attention: a page table row reaches %lld keys, at most 2^31 - 256", (long long)(table->shape[1] * k->shape[1]));
  if (q->shape[1] * q->shape[2] > 0x7fffffffll || q->shape[2] > 0x3fffffffll) return set_error(ctx, LH_ERR_UNSUPPORTED, "paged_attention: too many query rows");
  return LH_OK;
}

int64_t simt_ctas(const lh_ctx* ctx) { return static_cast<int64_t>(ctx->sm_count) * SIMT_CTAS_PER_SM; }

}  // namespace
}  // namespace lh

using namespace lh;

extern "C" int lh_b200_paged_append(lh_ctx_t* ctx, const lh_memref_t* q, const lh_memref_t* k, const lh_memref_t* v, const lh_memref_t* k_pages,
                                    const lh_memref_t* v_pages, const lh_memref_t* slots, const lh_memref_t* positions, float theta) {
  if (!ctx) return LH_ERR_INVALID;
  if (!k || !v || !k_pages || !v_pages || !slots) return set_error(ctx, LH_ERR_INVALID, "paged_append: k, v, k_pages, v_pages and slots are required");
  if (k->rank != 3 || v->rank != 3 || (q && q->rank != 3)) return set_error(ctx, LH_ERR_INVALID, "paged_append: q, k and v are rank-3 (tokens, heads, D) views");
  if (k_pages->rank != 4 || v_pages->rank != 4) return set_error(ctx, LH_ERR_INVALID, "paged_append: k_pages and v_pages are rank-4 (pages, page_size, Hkv, D) views");
  if (slots->rank != 1 || (positions && positions->rank != 1)) return set_error(ctx, LH_ERR_INVALID, "paged_append: slots and positions are (tokens)");
  for (const lh_memref_t* m : {q, k, v, k_pages, v_pages, slots, positions})
    if (m && !sane_extents(m)) return set_error(ctx, LH_ERR_INVALID, "paged_append: extent out of range");
  for (int i = 0; i < 3; ++i)
    if (v->shape[i] != k->shape[i]) return set_error(ctx, LH_ERR_INVALID, "paged_append: v must have k's shape");
  for (int i = 0; i < 4; ++i)
    if (v_pages->shape[i] != k_pages->shape[i]) return set_error(ctx, LH_ERR_INVALID, "paged_append: v_pages must have k_pages's shape");
  const int64_t T = k->shape[0], D = k->shape[2];
  if (k_pages->shape[2] != k->shape[1] || k_pages->shape[3] != D || D < 1 || k->shape[1] < 1) return set_error(ctx, LH_ERR_INVALID, "paged_append: the pages hold %lld heads of %lld, k has %lld of %lld", (long long)k_pages->shape[2], (long long)k_pages->shape[3], (long long)k->shape[1], (long long)D);
  if (k_pages->shape[1] < 1) return set_error(ctx, LH_ERR_INVALID, "paged_append: page size must be at least 1");
  if (q && (q->shape[0] != T || q->shape[2] != D)) return set_error(ctx, LH_ERR_INVALID, "paged_append: q must have k's tokens and head size");
  if (slots->shape[0] != T || (positions && positions->shape[0] != T)) return set_error(ctx, LH_ERR_INVALID, "paged_append: slots and positions must have one entry per token");
  const bool rotate = theta != 0.f;
  if (rotate && !(theta > 0.f && theta < INFINITY)) return set_error(ctx, LH_ERR_INVALID, "paged_append: theta must be positive and finite, or 0 for no rotation");
  if (rotate && !positions) return set_error(ctx, LH_ERR_INVALID, "paged_append: a rotation needs positions");
  if (rotate && D % 2) return set_error(ctx, LH_ERR_UNSUPPORTED, "paged_append: the head size must be even to rotate");
  if (D > 2 * APPEND_MAX_PAIRS) return set_error(ctx, LH_ERR_UNSUPPORTED, "paged_append: head size %lld is above %d", (long long)D, 2 * APPEND_MAX_PAIRS);
  if (!float_type(k->dtype) || !float_type(k_pages->dtype)) return set_error(ctx, LH_ERR_UNSUPPORTED, "paged_append: f32, bf16 or f16 operands");
  if (v->dtype != k->dtype || (q && q->dtype != k->dtype) || v_pages->dtype != k_pages->dtype) return set_error(ctx, LH_ERR_INVALID, "paged_append: q, k and v must have one type, and so must the pages");
  for (const lh_memref_t* m : {slots, positions})
    if (m && m->dtype != LH_I32 && m->dtype != LH_I64) return set_error(ctx, LH_ERR_INVALID, "paged_append: slots and positions are i32 or i64");
  for (const lh_memref_t* m : {q, k, v, k_pages, v_pages})
    if (m && D > 1 && m->strides[m->rank - 1] != 1) return set_error(ctx, LH_ERR_UNSUPPORTED, "paged_append: the head dimension must have unit stride");
  for (const lh_memref_t* m : {q, k_pages, v_pages})
    if (m && overlaps_itself(m)) return set_error(ctx, LH_ERR_INVALID, "paged_append: a written operand overlaps itself (zero stride)");
  const int64_t Hq = q ? q->shape[1] : 0;
  if ((Hq + 2 * k->shape[1]) * D > 0x7fffffffll) return set_error(ctx, LH_ERR_UNSUPPORTED, "paged_append: a token's rows are too long");
  if (T == 0) return LH_OK;
  AppendParams p;
  memset(&p, 0, sizeof(p));
  if (q) { p.q = data_ptr(q); p.sqt = q->strides[0]; p.sqh = q->strides[1]; }
  p.k = data_ptr(k); p.skt = k->strides[0]; p.skh = k->strides[1];
  p.v = data_ptr(v); p.svt = v->strides[0]; p.svh = v->strides[1];
  p.kp = data_ptr(k_pages); p.kpp = k_pages->strides[0]; p.kps = k_pages->strides[1]; p.kph = k_pages->strides[2];
  p.vp = data_ptr(v_pages); p.vpp = v_pages->strides[0]; p.vps = v_pages->strides[1]; p.vph = v_pages->strides[2];
  p.slots = data_ptr(slots); p.sslot = slots->strides[0]; p.slots64 = slots->dtype == LH_I64;
  if (positions) { p.pos = data_ptr(positions); p.spos = positions->strides[0]; p.pos64 = positions->dtype == LH_I64; }
  p.num_slots = k_pages->shape[0] * k_pages->shape[1];
  p.Hq = static_cast<int>(Hq); p.Hkv = static_cast<int>(k->shape[1]); p.D = static_cast<int>(D); p.page = static_cast<int>(k_pages->shape[1]);
  p.q_dtype = k->dtype; p.c_dtype = k_pages->dtype;
  p.rotate = rotate;
  p.log2_theta = rotate ? log2(static_cast<double>(theta)) : 0.0;
  p.dev_status = ctx->dev_status;
  // eight elements of every operand at a 16-byte boundary (32 for f32, read as two)
  bool vec = D % 8 == 0;
  for (const lh_memref_t* m : {q, k, v, k_pages, v_pages}) {
    if (!m || !vec) continue;
    vec = reinterpret_cast<uintptr_t>(data_ptr(m)) % 16 == 0;
    for (int i = 0; i + 1 < m->rank; ++i)
      if (m->shape[i] > 1 && m->strides[i] * static_cast<int64_t>(dtype_size(m->dtype)) % 16) vec = false;
  }
  const int64_t units = (Hq + 2 * k->shape[1]) * (vec ? D / 8 : (D + 1) / 2);
  // A few tokens do not fill the GPU with one CTA each: spread a token's rows over several, so
  // that every thread has one unit. They repeat the angles, which costs nothing on idle SMs.
  int64_t split = (units + APPEND_THREADS - 1) / APPEND_THREADS;
  if (T * split > static_cast<int64_t>(ctx->sm_count) * 8) split = 1;
  if (split > 65535) split = 65535;
  DeviceScope scope(ctx->device);
  AppendKernel kernel = vec ? append_vec_for(p.q_dtype, p.c_dtype) : append_generic_kernel;
  kernel<<<dim3(static_cast<unsigned>(T), static_cast<unsigned>(split)), APPEND_THREADS, 0, ctx->stream>>>(p);
  LH_CHECK_LAUNCH(ctx, "append_kernel");
  return LH_OK;
}

extern "C" int lh_b200_paged_attention_workspace(lh_ctx_t* ctx, const lh_memref_t* q, const lh_memref_t* k_pages, size_t* bytes) {
  if (!ctx) return LH_ERR_INVALID;
  if (!q || !k_pages || !bytes || q->rank != 4 || k_pages->rank != 4 || k_pages->shape[2] < 1) return set_error(ctx, LH_ERR_INVALID, "paged_attention_workspace: q (B, Hq, S, D), k_pages (pages, page_size, Hkv, D) and bytes are required");
  // enough for whichever kernel the operands' alignment selects
  const int Dp = static_cast<int>((q->shape[3] + 3) / 4 * 4);
  const int64_t rows = q->shape[1] / k_pages->shape[2] * q->shape[2];
  const size_t simt = workspace_for(simt_ctas(ctx), SIMT_ROWS, Dp).bytes;
  const int D = q->shape[3] > 256 ? 256 : static_cast<int>(q->shape[3]);
  const size_t mma = workspace_for(paged_mma_ctas(ctx, D), paged_mma_unit_rows(rows, D), Dp).bytes;
  *bytes = simt > mma ? simt : mma;
  return LH_OK;
}

extern "C" int lh_b200_paged_attention(lh_ctx_t* ctx, const lh_memref_t* o, const lh_memref_t* q, const lh_memref_t* k_pages, const lh_memref_t* v_pages,
                                       const lh_memref_t* page_table, const lh_memref_t* lengths, const lh_memref_t* workspace, float scale) {
  if (!ctx) return LH_ERR_INVALID;
  int rc = check_attention(ctx, o, q, k_pages, v_pages, page_table, lengths);
  if (rc) return rc;
  size_t need = 0;
  rc = lh_b200_paged_attention_workspace(ctx, q, k_pages, &need);
  if (rc) return rc;
  if (!workspace) return set_error(ctx, LH_ERR_INVALID, "paged_attention: a workspace is required");
  if (!is_contiguous(workspace) || reinterpret_cast<uintptr_t>(data_ptr(workspace)) % 256) return set_error(ctx, LH_ERR_INVALID, "paged_attention: the workspace must be contiguous and 256-byte aligned");
  const size_t have = static_cast<size_t>(numel(workspace)) * dtype_size(workspace->dtype);
  if (have < need) return set_error(ctx, LH_ERR_NOMEM, "paged_attention: the workspace holds %zu bytes, %zu are needed (lh_b200_paged_attention_workspace)", have, need);
  if (q->shape[0] == 0 || q->shape[1] == 0 || q->shape[2] == 0) return LH_OK;
  PagedParams p;
  memset(&p, 0, sizeof(p));
  p.q = data_ptr(q); p.sqb = q->strides[0]; p.sqh = q->strides[1]; p.sqs = q->strides[2];
  p.o = data_ptr(o); p.sob = o->strides[0]; p.soh = o->strides[1]; p.sos = o->strides[2];
  p.k = data_ptr(k_pages); p.skp = k_pages->strides[0]; p.sks = k_pages->strides[1]; p.skh = k_pages->strides[2];
  p.v = data_ptr(v_pages); p.svp = v_pages->strides[0]; p.svs = v_pages->strides[1]; p.svh = v_pages->strides[2];
  p.table = static_cast<const int*>(static_cast<void*>(data_ptr(page_table))); p.stb = page_table->strides[0]; p.stp = page_table->strides[1];
  p.lengths = static_cast<const int*>(static_cast<void*>(data_ptr(lengths))); p.slen = lengths->strides[0];
  p.num_pages = k_pages->shape[0];
  p.B = static_cast<int>(q->shape[0]); p.Hkv = static_cast<int>(k_pages->shape[2]); p.group = static_cast<int>(q->shape[1] / k_pages->shape[2]);
  p.Sq = static_cast<int>(q->shape[2]); p.D = static_cast<int>(q->shape[3]);
  p.page = static_cast<int>(k_pages->shape[1]);
  p.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (p.page == 1 << s) p.page_shift = s;
  p.max_keys = static_cast<int>(page_table->shape[1] * k_pages->shape[1]);
  p.rows = p.group * p.Sq;
  p.o_dtype = o->dtype;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.Dp = (p.D + 3) / 4 * 4;
  p.dev_status = ctx->dev_status;
  const bool mma = paged_mma_supported(k_pages, v_pages);
  p.unit_rows = mma ? paged_mma_unit_rows(p.rows, p.D) : SIMT_ROWS;
  p.tile = SIMT_TILE;
  const int ctas = static_cast<int>(mma ? paged_mma_ctas(ctx, p.D) : simt_ctas(ctx));
  p.row_groups = (p.rows + p.unit_rows - 1) / p.unit_rows;
  if (static_cast<int64_t>(p.Hkv) * p.row_groups > 0x7fffffffll) return set_error(ctx, LH_ERR_UNSUPPORTED, "paged_attention: too many query rows");
  const Workspace w = workspace_for(ctas, p.unit_rows, p.Dp);
  char* base = data_ptr(workspace);
  p.total = reinterpret_cast<int64_t*>(base);
  p.first = reinterpret_cast<int4*>(base + w.first);
  p.ml = reinterpret_cast<float2*>(base + w.ml);
  p.part = reinterpret_cast<float*>(base + w.part);
  DeviceScope scope(ctx->device);
  if (mma) {
    rc = paged_mma_launch(ctx, p, q->dtype, ctas);
    if (rc) return rc;
    return join_launch(ctx, p, ctas);
  }
  const bool vec = p.D % 4 == 0 && aligned_view(k_pages, 4) && aligned_view(v_pages, 4);
  PagedKernel kernel = q->dtype == LH_F32 ? simt_kernel_for<float>(p.D, vec) : q->dtype == LH_BF16 ? simt_kernel_for<__nv_bfloat16>(p.D, vec) : simt_kernel_for<__half>(p.D, vec);
  kernel<<<static_cast<unsigned>(ctas), SIMT_THREADS, 0, ctx->stream>>>(p);
  LH_CHECK_LAUNCH(ctx, "paged_simt_kernel");
  return join_launch(ctx, p, ctas);
}
