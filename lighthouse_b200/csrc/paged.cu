// The paged key-value cache: writing new rows into it (rotary embedding fused in) and
// attending over it. Entry points lh_b200_paged_append, lh_b200_paged_attention.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace lh {
namespace {

// ------------------------------------------------------------------- append
// For token t: q <- rot(q, pos[t]) in place, page rows of slot[t] <- rot(k, pos[t]) and v.
// A pure copy: bound by the bytes of q (twice), k, v and their cache rows, and for a few
// tokens by latency. One CTA (or several, below) per token: the D/2 angles are computed once
// into shared memory and used by every head. 12289 tokens of 32 + 2 x 8 heads of 128 in f32 (f16 pages)
// take 88 us, 6.0 TB/s; 1 to 256 tokens 6.4 us, a launch.
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
// The general kernel, on FFMA: f32 caches, and 16-bit ones whose rows are not 16-byte aligned. For
// f32 with four query rows to a kv head it needs 512 FFMA and about 450 shared-memory wavefronts
// per 16 keys of D = 128 (16 KB), two thirds of what an SM has time for while those bytes arrive. 64
// sequences of up to 4096 keys (16 heads on 4) take 153 us, 3.6 TB/s; 8 of them 48 us, of which
// about 20 are what any call takes (start, lengths, pages, join) and 11 the join of its parts. (Four
// warps an SM with three stages each took 50; two more warps' chains of loads, products and
// softmax overlap for the same bytes in flight.)
// A warp fetches 16 keys at a time into a ring of f32 rows (cp.async; or, ASYNC false, loads and
// conversions of single elements). Scores: a lane has four keys and an eighth of their dimensions, so
// that a load of Q serves four keys and one of K all rows; the eighths are then added up in halving
// steps, after which a lane has one key and half of the rows. P V: a lane has four dimensions (of
// 64 only half the lanes' worth: the halves take alternate keys).
constexpr int SIMT_ROWS = 8;

template <int DP>
struct SimtShape {
  static constexpr int warps = DP == 256 ? 3 : 6;
  static constexpr int stages = 2;
  static constexpr int stage_floats = 2 * TILE * DP;  // K and V rows of 16 keys
  static constexpr int ctas_per_sm = DP == 64 ? 2 : 1;
  static constexpr int q_pitch = DP;
  template <int R>
  static constexpr int warp_floats() { return stages * stage_floats + R * q_pitch + TILE * R; }
  template <int R>
  static constexpr int smem() { return warps * warp_floats<R>() * 4; }
};

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  if constexpr (std::is_same<T, float>::value) return x;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
  else return __bfloat162float(x);
}

template <typename T, int DP, int R, bool ASYNC>
__global__ void __launch_bounds__(SimtShape<DP>::warps * 32, SimtShape<DP>::ctas_per_sm) paged_simt_kernel(const PagedParams p) {
  using S = SimtShape<DP>;
  constexpr int THREADS = S::warps * 32, CHUNKS = DP / 4;
  constexpr int RH = R / 2;  // rows of which a lane has the scores
  constexpr int NV = DP == 256 ? 2 : 1, AT_ONCE = DP == 64 ? 2 : 1;  // P V: vectors of a lane, keys taken at once
  extern __shared__ __align__(16) float ring_mem[];
  __shared__ uint32_t there[S::warps][S::stages];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_dependency_trigger();
  TileCursor at;
  int64_t left = find_stretch<THREADS>(p, at);
  if (left == 0) return;
  float* const ring = ring_mem + warp * S::template warp_floats<R>();
  float* const qs = ring + S::stages * S::stage_floats;
  float* const ps = qs + R * S::q_pitch;
  const T* const K = static_cast<const T*>(p.k);
  const T* const V = static_cast<const T*>(p.v);

  Fetch f;
  f.at = at;
  f.left = left;
  f.look_up(p, lane & 15);
  auto fetch = [&](int stage) {
    if (f.left <= 0) return;
    const int key0 = f.at.t * TILE, hkv = f.at.u / p.row_groups;
    const int j = key0 + (lane & 15);
    const bool live = j < f.at.len, inside = f.page_id >= 0 && f.page_id < p.num_pages;
    if (live && !inside) report_bad_index(p.dev_status);
    const uint32_t mask = __ballot_sync(0xffffffffu, live && inside) & 0xffffu;
    const int slot = j - page_of(p, j) * p.page;
    const int64_t ko = live && inside ? f.page_id * p.skp + slot * p.sks + hkv * p.skh : 0;
    const int64_t vo = live && inside ? f.page_id * p.svp + slot * p.svs + hkv * p.svh : 0;
    float* const to = ring + stage * S::stage_floats;
    if (mask) {
#pragma unroll 8
      for (int i = 0; i < TILE * CHUNKS / 32; ++i) {
        const int row = (i * 32 + lane) / CHUNKS, chunk = (i * 32 + lane) % CHUNKS;
        const int64_t kr = __shfl_sync(0xffffffffu, ko, row), vr = __shfl_sync(0xffffffffu, vo, row);
        const int d = chunk * 4;
        const bool get = (mask >> row & 1) && d < p.D;
        float* const dst = to + row * DP + ((chunk ^ (row & 7)) << 2);
        if constexpr (ASYNC) {
          const uint32_t s = smem_u32(dst);
          cp_async16(s, get ? K + kr + d : K, get ? 16 : 0);
          cp_async16(s + TILE * DP * 4, get ? V + vr + d : V, get ? 16 : 0);
        } else {
          float k4[4], v4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool one = get && d + e < p.D;
            k4[e] = one ? to_f32(K[kr + d + e]) : 0.f;
            v4[e] = one ? to_f32(V[vr + d + e]) : 0.f;
          }
          *reinterpret_cast<float4*>(dst) = make_float4(k4[0], k4[1], k4[2], k4[3]);
          *reinterpret_cast<float4*>(dst + TILE * DP) = make_float4(v4[0], v4[1], v4[2], v4[3]);
        }
      }
    }
    if (lane == 0) there[warp][stage] = mask;
    f.advance(p);
    f.look_up(p, lane & 15);
  };
#pragma unroll
  for (int s = 0; s < S::stages; ++s) {
    fetch(s);
    cp_async_commit();
  }

  const int eighth = lane & 7, key4 = (lane >> 3) * 4;      // of the products
  const int key = key4 + (eighth >> 1), rows0 = (lane & 1) * RH;  // of the scores
  const int half = lane >> 4;
  const int my_chunk = DP == 64 ? lane & 15 : lane;  // P V
  float m[RH], l[RH], acc[R][NV * 4];
  int seen[RH];
  int t0 = at.t, stage = 0;
  bool fresh = true;
  for (; left > 0; --left) {
    const int hkv = at.u / p.row_groups, row0 = (at.u % p.row_groups) * R;
    const int nrows = min(R, p.rows - row0);
    if (fresh) {
      fresh = false;
      t0 = at.t;
      __syncwarp();
      constexpr int TOGETHER = R * DP / 32 < 16 ? R * DP / 32 : 16;  // loads on their way at a time
#pragma unroll 1
      for (int i0 = lane; i0 < R * DP; i0 += 32 * TOGETHER) {
        float x[TOGETHER];
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k) {
          const int r = (i0 + k * 32) / DP, d = (i0 + k * 32) % DP;
          x[k] = r < nrows && d < p.D ? to_f32(static_cast<const T*>(p.q)[at.b * p.sqb + row_head(p, hkv, row0 + r) * p.sqh + row_token(p, row0 + r) * p.sqs + d]) * p.scale_log2 : 0.f;
        }
#pragma unroll
        for (int k = 0; k < TOGETHER; ++k) {
          const int r = (i0 + k * 32) / DP, d = (i0 + k * 32) % DP;
          qs[r * S::q_pitch + d] = x[k];
        }
      }
#pragma unroll
      for (int r = 0; r < RH; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
        seen[r] = rows0 + r < nrows ? at.len - p.Sq + 1 + row_token(p, row0 + rows0 + r) : 0;  // keys that the row may attend to
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int i = 0; i < NV * 4; ++i) acc[r][i] = 0.f;
      }
    }
    cp_async_wait<S::stages - 1>();
    __syncwarp();
    const uint32_t mask = there[warp][stage];
    if (mask) {
      const float* const kt = ring + stage * S::stage_floats;
      const float* const vt = kt + TILE * DP;
      const int key0 = at.t * TILE;
      float part[R][4];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < 4; ++k) part[r][k] = 0.f;
#pragma unroll
      for (int c = 0; c < CHUNKS / 8; ++c) {
        float4 kv[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) kv[k] = *reinterpret_cast<const float4*>(kt + (key4 + k) * DP + (((c * 8 + eighth) ^ ((key4 + k) & 7)) << 2));
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float4 qv = *reinterpret_cast<const float4*>(qs + r * S::q_pitch + (c * 8 + eighth) * 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) part[r][k] = fmaf(qv.x, kv[k].x, fmaf(qv.y, kv[k].y, fmaf(qv.z, kv[k].z, fmaf(qv.w, kv[k].w, part[r][k]))));
        }
      }
      // Each step gives half of what is left to the lane across and adds what comes back: keys 2 and 3 against 0
      // and 1, then the odd key, then the second half of the rows.
      float two[R][2], one[R], s[RH];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float give = lane & 4 ? part[r][k] : part[r][k + 2];
          two[r][k] = (lane & 4 ? part[r][k + 2] : part[r][k]) + __shfl_xor_sync(0xffffffffu, give, 4);
        }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float give = lane & 2 ? two[r][0] : two[r][1];
        one[r] = (lane & 2 ? two[r][1] : two[r][0]) + __shfl_xor_sync(0xffffffffu, give, 2);
      }
#pragma unroll
      for (int r = 0; r < RH; ++r) {
        const float give = lane & 1 ? one[r] : one[r + RH];
        s[r] = (lane & 1 ? one[r + RH] : one[r]) + __shfl_xor_sync(0xffffffffu, give, 1);
      }
      // keys that only the later of several new tokens may see: masked rows must not meet their V
      const bool partial = key0 + TILE > at.len - p.Sq + 1;
      bool grows = false;
#pragma unroll
      for (int r = 0; r < RH; ++r) {
        if (!(mask >> key & 1) || key0 + key >= seen[r]) s[r] = -INFINITY;
        grows |= s[r] > m[r];
      }
      // the running maximum is only brought up to date when some key passes it
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int r = 0; r < RH; ++r) {
          float top = s[r];
#pragma unroll
          for (int d = 2; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          top = fmaxf(top, m[r]);
          const float alpha = top == -INFINITY ? 1.f : exp2f(m[r] - top), others = __shfl_xor_sync(0xffffffffu, alpha, 1);
          m[r] = top;
          l[r] *= alpha;
#pragma unroll
          for (int i = 0; i < NV * 4; ++i) {
            acc[r][i] *= lane & 1 ? others : alpha;
            acc[r + RH][i] *= lane & 1 ? alpha : others;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < RH; ++r) {
        const float e = exp2_safe(s[r], m[r]);
        l[r] += e;
        ps[key * R + rows0 + r] = e;
      }
      __syncwarp();
#pragma unroll 4
      for (int j0 = 0; j0 < TILE; j0 += AT_ONCE) {
        const int j = AT_ONCE == 2 ? j0 + half : j0;
        float e[R];
#pragma unroll
        for (int r = 0; r < R; ++r) e[r] = ps[j * R + r];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const float4 vv = *reinterpret_cast<const float4*>(vt + j * DP + (((my_chunk + i * 32) ^ (j & 7)) << 2));
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (partial && e[r] == 0.f) continue;
            acc[r][i * 4 + 0] = fmaf(e[r], vv.x, acc[r][i * 4 + 0]);
            acc[r][i * 4 + 1] = fmaf(e[r], vv.y, acc[r][i * 4 + 1]);
            acc[r][i * 4 + 2] = fmaf(e[r], vv.z, acc[r][i * 4 + 2]);
            acc[r][i * 4 + 3] = fmaf(e[r], vv.w, acc[r][i * 4 + 3]);
          }
        }
      }
    }
    __syncwarp();
    if (++at.t == at.tiles || left == 1) {
      // ---- the warp leaves the unit
      const int64_t slot = partial_slot<THREADS>(t0, at.t, at.tiles);
      float m_of[R], l_of[R];
#pragma unroll
      for (int r = 0; r < RH; ++r) {
#pragma unroll
        for (int d = 2; d < 32; d <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
        const float m_other = __shfl_xor_sync(0xffffffffu, m[r], 1), l_other = __shfl_xor_sync(0xffffffffu, l[r], 1);
        m_of[r] = lane & 1 ? m_other : m[r];
        m_of[r + RH] = lane & 1 ? m[r] : m_other;
        l_of[r] = lane & 1 ? l_other : l[r];
        l_of[r + RH] = lane & 1 ? l[r] : l_other;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (AT_ONCE == 2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][i] += __shfl_xor_sync(0xffffffffu, acc[r][i], 16);
        }
        if (r >= nrows) continue;
        const float inv = l_of[r] == 0.f ? 0.f : 1.f / l_of[r];  // a row that sees no key has no weight: zeros
        const int64_t out = at.b * p.sob + row_head(p, hkv, row0 + r) * p.soh + row_token(p, row0 + r) * p.sos;
        if (slot >= 0 && lane == 0) p.ml[slot * p.part_rows + r] = make_float2(m_of[r], l_of[r]);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int d = (my_chunk + i * 32) * 4;
          if (DP == 64 && lane >= 16) break;
          float4 v = make_float4(acc[r][i * 4], acc[r][i * 4 + 1], acc[r][i * 4 + 2], acc[r][i * 4 + 3]);
          if (slot < 0) {
            v.x *= inv; v.y *= inv; v.z *= inv; v.w *= inv;
            store_o4(p, out, d, v);
          } else if (d < p.Dp) {
            *reinterpret_cast<float4*>(p.part + (slot * p.part_rows + r) * p.Dp + d) = v;
          }
        }
      }
      fresh = true;
      if (left > 1) at.next_unit(p);
    }
    fetch(stage);
    cp_async_commit();
    stage = stage + 1 == S::stages ? 0 : stage + 1;
  }
}

// Joins the units that several warps worked on: each warp of the join looks at one border between two
// stretches, and if that is the first border inside a unit, the unit's parts are added up: by the
// warp itself when they are few, else by its whole block (the warps take the parts in turn, a lane
// holds four head dimensions). The stretches fix the order of every sum. The kernel also writes the
// zeros of sequences that hold no keys. It is a programmatic dependent of the kernel above: resident
// and waiting when that one ends.
struct JoinWork {
  int parts;   // 0: nothing to join at this border
  int b, u;
  int64_t c0;  // the first part's stretch
};

__device__ __forceinline__ int64_t join_slot(const JoinWork& w, int c) { return c == 0 ? 2 * w.c0 + 1 : 2 * (w.c0 + c); }

__global__ void __launch_bounds__(JOIN_WARPS * 32, 4) paged_join_kernel(const PagedParams p, int64_t stretches) {
  __shared__ JoinWork work[JOIN_WARPS];
  __shared__ float red[JOIN_WARPS];
  __shared__ float4 sums[JOIN_WARPS][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int ALONE = 32;  // parts that a warp adds up by itself
  grid_dependency_wait();
  if (blockIdx.y == 0) {
    const int64_t per = static_cast<int64_t>(p.Hkv) * p.group * p.Sq * p.D;
    for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
      if (paged_length(p, b)) continue;
      for (int64_t i = tid; i < per; i += JOIN_WARPS * 32) {
        const int d = static_cast<int>(i % p.D);
        const int64_t rest = i / p.D;
        store_from_f32(p.o, p.o_dtype, b * p.sob + (rest / p.Sq) * p.soh + (rest % p.Sq) * p.sos + d, 0.f);
      }
    }
  }
  const int64_t i = static_cast<int64_t>(blockIdx.x) * JOIN_WARPS + warp;
  JoinWork w = {0, 0, 0, 0};
  if (i > 0 && i < stretches) {
    const int4 here = p.first[i];  // the unit's tiles with it: nothing to look up in turn
    const int64_t total = *p.total;
    if (here.x >= 0 && here.z > 0) {  // a stretch that begins inside its unit
      const int64_t n = stretch_count(total, stretches);
      const int64_t begin = stretch_begin(total, n, i) - here.z;  // the unit's first tile
      if (stretch_begin(total, n, i - 1) <= begin) {  // no earlier border lies in this unit
        const int64_t end = begin + here.w;
        w.c0 = i - 1;
        w.parts = static_cast<int>(stretch_owner(total, n, end - 1) - w.c0 + 1);
        w.b = here.x;
        w.u = here.y;
      }
    }
  }
  if (lane == 0) work[warp] = w;
  if (w.parts && w.parts <= ALONE) {
    const int hkv = w.u / p.row_groups, row0 = (w.u % p.row_groups) * p.unit_rows;
    const int nrows = min(p.unit_rows, p.rows - row0);
    for (int r = blockIdx.y; r < nrows; r += gridDim.y) {
      const float2 mine = lane < w.parts ? p.ml[join_slot(w, lane) * p.part_rows + r] : make_float2(-INFINITY, 0.f);
      float M = mine.x;
#pragma unroll
      for (int d = 16; d; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
      const float scale = exp2_safe(mine.x, M);
      float L = mine.y * scale;
#pragma unroll
      for (int d = 16; d; d >>= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
      const float inv = L == 0.f ? 0.f : 1.f / L;  // a row that sees no key has no weight: zeros
      const int row = row0 + r;
      const int64_t out = w.b * p.sob + row_head(p, hkv, row) * p.soh + row_token(p, row) * p.sos;
      for (int d0 = 0; d0 < p.Dp; d0 += 128) {
        const int d = d0 + lane * 4;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        // parts lie two slots apart, but for the first; six of them are on their way at a time
        const int64_t apart = 2 * static_cast<int64_t>(p.part_rows) * p.Dp;
        const float* const first = p.part + (join_slot(w, 0) * p.part_rows + r) * p.Dp + (d < p.Dp ? d : 0);
        const float* const rest = first - apart / 2;
        constexpr int BATCH = 6;
        for (int c0 = 0; c0 < w.parts; c0 += BATCH) {
          float4 x[BATCH];
#pragma unroll
          for (int c = 0; c < BATCH; ++c) x[c] = *reinterpret_cast<const float4*>(c0 + c == 0 ? first : rest + min(c0 + c, w.parts - 1) * apart);
#pragma unroll
          for (int c = 0; c < BATCH; ++c) {
            const float k = __shfl_sync(0xffffffffu, scale, min(c0 + c, 31));
            if (c0 + c < w.parts) {
              a.x = fmaf(x[c].x, k, a.x); a.y = fmaf(x[c].y, k, a.y); a.z = fmaf(x[c].z, k, a.z); a.w = fmaf(x[c].w, k, a.w);
            }
          }
        }
        store_o4(p, out, d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
      }
    }
  }
  if (!__syncthreads_or(w.parts > ALONE)) return;
  for (int q = 0; q < JOIN_WARPS; ++q) {
    w = work[q];
    if (w.parts <= ALONE) continue;
    const int hkv = w.u / p.row_groups, row0 = (w.u % p.row_groups) * p.unit_rows;
    const int nrows = min(p.unit_rows, p.rows - row0);
    for (int r = blockIdx.y; r < nrows; r += gridDim.y) {
      float M = -INFINITY;
      for (int c = tid; c < w.parts; c += JOIN_WARPS * 32) M = fmaxf(M, p.ml[join_slot(w, c) * p.part_rows + r].x);
#pragma unroll
      for (int d = 16; d; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
      if (lane == 0) red[warp] = M;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < JOIN_WARPS; ++k) M = fmaxf(M, red[k]);
      const int row = row0 + r;
      const int64_t out = w.b * p.sob + row_head(p, hkv, row) * p.soh + row_token(p, row) * p.sos;
      for (int d0 = 0; d0 < p.Dp; d0 += 128) {
        const int d = d0 + lane * 4;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        float L = 0.f;
#pragma unroll 8
        for (int c = warp; c < w.parts; c += JOIN_WARPS) {
          const int64_t from = join_slot(w, c) * p.part_rows + r;
          const float2 ml = p.ml[from];
          const float k = exp2_safe(ml.x, M);
          L = fmaf(ml.y, k, L);
          if (d < p.Dp) {
            const float4 x = *reinterpret_cast<const float4*>(p.part + from * p.Dp + d);
            a.x = fmaf(x.x, k, a.x); a.y = fmaf(x.y, k, a.y); a.z = fmaf(x.z, k, a.z); a.w = fmaf(x.w, k, a.w);
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
          for (int k = 0; k < JOIN_WARPS; ++k) {
            const float4 x = sums[k][lane];
            a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
            L += red[k];
          }
          const float inv = L == 0.f ? 0.f : 1.f / L;
          store_o4(p, out, d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
        }
      }
      __syncthreads();
    }
  }
}

int join_launch(lh_ctx* ctx, const PagedParams& p, int64_t stretches) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  // rows side by side: a unit split over the whole GPU has many parts to each row
  cfg.gridDim = dim3(static_cast<unsigned>((stretches + JOIN_WARPS - 1) / JOIN_WARPS), static_cast<unsigned>(p.part_rows < 8 ? p.part_rows : 8));
  cfg.blockDim = dim3(JOIN_WARPS * 32);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LH_CUDA_CHECK(ctx, cudaLaunchKernelEx(&cfg, paged_join_kernel, p, stretches));
  LH_CHECK_LAUNCH(ctx, "paged_join_kernel");
  return LH_OK;
}

int simt_unit_rows(int64_t rows) { return rows <= 2 ? 2 : rows <= 4 ? 4 : SIMT_ROWS; }
int simt_stretches(const lh_ctx* ctx, int D) {
  return ctx->sm_count * (D <= 64 ? SimtShape<64>::warps * SimtShape<64>::ctas_per_sm : D <= 128 ? SimtShape<128>::warps * SimtShape<128>::ctas_per_sm : SimtShape<256>::warps * SimtShape<256>::ctas_per_sm);
}

template <typename T, int DP, int R, bool ASYNC>
int simt_launch(lh_ctx* ctx, const PagedParams& p, int stretches) {
  constexpr int smem = SimtShape<DP>::template smem<R>();
  auto* kernel = paged_simt_kernel<T, DP, R, ASYNC>;
  LH_CUDA_CHECK(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kernel<<<static_cast<unsigned>(stretches / SimtShape<DP>::warps), SimtShape<DP>::warps * 32, smem, ctx->stream>>>(p);
  LH_CHECK_LAUNCH(ctx, "paged_simt_kernel");
  return LH_OK;
}
template <typename T, int DP, bool ASYNC>
int simt_launch_rows(lh_ctx* ctx, const PagedParams& p, int stretches) {
  return p.unit_rows == 2 ? simt_launch<T, DP, 2, ASYNC>(ctx, p, stretches) : p.unit_rows == 4 ? simt_launch<T, DP, 4, ASYNC>(ctx, p, stretches) : simt_launch<T, DP, SIMT_ROWS, ASYNC>(ctx, p, stretches);
}
template <typename T, bool ASYNC>
int simt_launch_size(lh_ctx* ctx, const PagedParams& p, int stretches) {
  return p.D <= 64 ? simt_launch_rows<T, 64, ASYNC>(ctx, p, stretches) : p.D <= 128 ? simt_launch_rows<T, 128, ASYNC>(ctx, p, stretches) : simt_launch_rows<T, 256, ASYNC>(ctx, p, stretches);
}

bool aligned_view(const lh_memref_t* m, int elems) {
  if (reinterpret_cast<uintptr_t>(data_ptr(m)) % (elems * dtype_size(m->dtype))) return false;
  for (int i = 0; i + 1 < m->rank; ++i)
    if (m->shape[i] > 1 && m->strides[i] % elems) return false;
  return true;
}

bool aligned_to_type(const lh_memref_t* m) { return reinterpret_cast<uintptr_t>(data_ptr(m)) % dtype_size(m->dtype) == 0; }

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
Workspace workspace_for(int64_t stretches, int64_t rows, int Dp) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  Workspace w;
  w.first = 256;  // the tile count comes first
  w.ml = w.first + up(stretches * sizeof(int4));
  w.part = w.ml + up(2 * stretches * rows * sizeof(float2));
  w.bytes = w.part + up(2 * stretches * static_cast<size_t>(rows) * Dp * sizeof(float));
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
  for (const lh_memref_t* m : {o, q, k, v, table, lengths})
    if (!aligned_to_type(m)) return set_error(ctx, LH_ERR_INVALID, "paged_attention: an operand is not aligned to its type");
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
  for (const lh_memref_t* m : {q, k, v, k_pages, v_pages, slots, positions})
    if (m && !aligned_to_type(m)) return set_error(ctx, LH_ERR_INVALID, "paged_append: an operand is not aligned to its type");
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
  const int Dp = static_cast<int>((q->shape[3] + 3) / 4 * 4), D = q->shape[3] > 256 ? 256 : static_cast<int>(q->shape[3]);
  const int64_t rows = q->shape[1] / k_pages->shape[2] * q->shape[2];
  const size_t simt = workspace_for(simt_stretches(ctx, D), std::min<int64_t>(rows, simt_unit_rows(rows)), Dp).bytes;
  const size_t mma = workspace_for(paged_mma_stretches(ctx, rows, D), std::min<int64_t>(rows, paged_mma_unit_rows(rows, D)), Dp).bytes;
  *bytes = std::max(simt, mma);
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
  p.unit_rows = mma ? paged_mma_unit_rows(p.rows, p.D) : simt_unit_rows(p.rows);
  p.part_rows = std::min(p.rows, p.unit_rows);
  // A unit's Q and epilogue against a tile, measured inside the kernels: 2000 clocks to 1000 with eight
  // rows, 3800 to 1300 with more; the FFMA kernel's tiles take as long as its epilogue.
  p.unit_cost = !mma ? 1 : p.unit_rows == 8 ? 2 : 3;
  const int stretches = mma ? paged_mma_stretches(ctx, p.rows, p.D) : simt_stretches(ctx, p.D);
  p.o_vec = p.D % 4 == 0 && aligned_view(o, 4);
  p.q_pairs = dtype_size(q->dtype) == 2 && aligned_view(q, 2);
  p.row_groups = (p.rows + p.unit_rows - 1) / p.unit_rows;
  if (static_cast<int64_t>(p.Hkv) * p.row_groups > 0x7fffffffll) return set_error(ctx, LH_ERR_UNSUPPORTED, "paged_attention: too many query rows");
  const Workspace w = workspace_for(stretches, p.part_rows, p.Dp);
  char* base = data_ptr(workspace);
  p.total = reinterpret_cast<int64_t*>(base);
  p.first = reinterpret_cast<int4*>(base + w.first);
  p.ml = reinterpret_cast<float2*>(base + w.ml);
  p.part = reinterpret_cast<float*>(base + w.part);
  DeviceScope scope(ctx->device);
  if (mma) rc = paged_mma_launch(ctx, p, q->dtype, stretches);
  else if (q->dtype == LH_F32) rc = p.D % 4 == 0 && aligned_view(k_pages, 4) && aligned_view(v_pages, 4) ? simt_launch_size<float, true>(ctx, p, stretches) : simt_launch_size<float, false>(ctx, p, stretches);
  else rc = q->dtype == LH_BF16 ? simt_launch_size<__nv_bfloat16, false>(ctx, p, stretches) : simt_launch_size<__half, false>(ctx, p, stretches);
  return rc ? rc : join_launch(ctx, p, stretches);
}
