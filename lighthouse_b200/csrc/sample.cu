// Sampling a token per row of logits. Entry point lh_b200_sample.
//
// Weights are whole numbers: w = round(2^42 exp((x - max) / T)), formed in f64. Sums of them are
// exact, so they come out the same in whatever order threads and CTAs add them, and a
// drawn token does not depend on how the row was cut up. In f32 the running sum of 10^5 weights
// is off by 1e-7 of the total, and as many borders between tokens lie in it: one row in some
// hundreds would get another token than the definition gives.
//
// A row belongs to a cluster of CTAs and stays in their shared memory: it is read once. What top-k
// and top-p keep is always "the first so many in the order of falling logits, equal ones by
// rising index", so each is one border in that order. It is found by a histogram of the
// row over log2 of the weight (4096 bins of 1/93 octave): the bin that the border falls in
// holds a few dozen tokens, which are collected in one CTA and ranked against each other.
// Bins too full for that (rows of equal logits) are first split by further digits of the
// order itself. The CTAs talk through distributed shared memory.
#include <cooperative_groups.h>

#include "common.cuh"
#include "epilogue.cuh"

namespace cg = cooperative_groups;

namespace lh {
namespace {

struct SampleParams {
  const void* logits; int64_t row_stride; int dtype;
  int rows, vocab;
  int items;  // values per thread: a CTA has items * SAMPLE_THREADS of the row
  const float* uniform; int64_t su;
  const float* temperature; int64_t st;
  const void* top_k; int64_t sk; int k64;
  const float* top_p; int64_t sp;
  const float* min_p; int64_t sm;
  void* tokens; int64_t stok; int tok64;
  float* logprobs; int64_t slp;
};

typedef unsigned long long u64;

constexpr int WEIGHT_BITS = 42;
constexpr u64 WEIGHT_ONE = 1ull << WEIGHT_BITS;  // the largest weight
constexpr int INDEX_BITS = 20;
constexpr int64_t MAX_VOCAB = int64_t(1) << INDEX_BITS;  // 2^20 weights of 2^42 stay within 63 bits
constexpr int SAMPLE_THREADS = 512;
constexpr int WARPS = SAMPLE_THREADS / 32;
constexpr int MAX_CLUSTER = 8;
constexpr int BINS = 4096;
constexpr float BINS_PER_OCTAVE = 93.f;  // the last bin starts 44 octaves below the maximum: weights of zero
constexpr int LIST = SAMPLE_THREADS;

// Values in an order that whole numbers keep; NaN ranks with -inf, -0 with +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x == x)) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }
// Position in the order of falling logits and rising index: larger comes first, no two are equal.
__device__ __forceinline__ u64 order_of(float x, int i) { return (static_cast<u64>(key_of(x)) << INDEX_BITS) | (MAX_VOCAB - 1 - i); }
__device__ __forceinline__ int index_of(u64 order) { return static_cast<int>(MAX_VOCAB - 1 - (order & (MAX_VOCAB - 1))); }
__device__ __forceinline__ float logit_of(u64 order) { return value_of(static_cast<uint32_t>(order >> INDEX_BITS)); }

constexpr int TABLE = 256;

struct Weighing {
  float top;
  double top64, scale;   // row maximum; 256 log2(e) / T
  float bin_scale;       // bins per two units of logit
  const double* table;   // 2^(42 + i / 256)
  // 2^t = 2^(j / 256) (1 + (e^(f ln2 / 256) - 1)), 256 t = j + f, |f| <= 1/2: the series' fourth term
  // and on are below 2^-42. Adding 2^52 leaves the rounded whole number in the low bits.
  __device__ __forceinline__ u64 of(float x) const {
    const double y = x == top ? 0.0 : (static_cast<double>(x) - top64) * scale;
    if (!(y > -(WEIGHT_BITS + 1.0) * TABLE)) return 0;  // also NaN, and (-inf) * 0
    const double magic = 6755399441055744.0;  // 1.5 * 2^52
    const double z = y + magic;
    const int j = __double2loint(z);
    const double f = y - (z - magic);
    const double a1 = 0.69314718055994530942 / TABLE;
    const double s = f * fma(f, fma(f, a1 * a1 * a1 / 6, a1 * a1 / 2), a1);
    const double base = table[j & (TABLE - 1)];
    const double scaled = __hiloint2double(__double2hiint(base) + (j >> 8) * (1 << 20), __double2loint(base));
    const double fixed = fma(scaled, s, scaled) + 4503599627370496.0;
    return static_cast<u64>(__double_as_longlong(fixed)) & ((1ull << 52) - 1);
  }
  // Falls with x. The last bin is for weights of zero. (Halves: the difference stays finite.)
  __device__ __forceinline__ int bin_of(float x) const {
    return x == top ? 0 : static_cast<int>(fminf((0.5f * top - 0.5f * x) * bin_scale, static_cast<float>(BINS - 1)));  // NaN: the last
  }
};

template <typename V>
__device__ __forceinline__ V warp_total(V v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

struct SampleShared {
  double table[TABLE];
  u64 hist[BINS];
  u64 list[LIST], mass[LIST];
  u64 from[4][MAX_CLUSTER];  // what each CTA of the cluster sent, per use
  u64 red[WARPS];
  u64 border, above;         // answers of the first CTA
  int bin, listed;
  int found;
};

// One CTA's part of a row. HELD: its values lie in shared memory; otherwise each pass reads them
// from global memory again (from L2: a cluster's row is in use by nobody else).
template <bool HELD>
struct Row {
  const float* held;
  const void* logits; int dtype; int64_t base;
  int offset, first, steps, vocab;  // this lane's place in the CTA's part and in the row, how many values it has (32 apart)
  __device__ __forceinline__ float value(int j) const {
    return HELD ? held[offset + j * 32] : load_as_f32(logits, dtype, base + first + j * 32);
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 4
    for (int j = 0; j < steps; ++j) {
      const int i = first + j * 32;
      if (i < vocab) f(value(j), i);
    }
  }
};

__device__ __forceinline__ u64 block_total(u64 v, u64* red) {
  v = warp_total(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) v += red[w];
  return v;
}

// Every CTA's value reaches every CTA; `use` numbers the exchanges of a row.
__device__ __forceinline__ void exchange(const cg::cluster_group& cluster, SampleShared& sh, int use, u64 v) {
  const unsigned n = cluster.num_blocks();
  if (threadIdx.x < n) cluster.map_shared_rank(&sh.from[use][cluster.block_rank()], threadIdx.x)[0] = v;
  cluster.sync();
}

// The border of a filter: the `want`-th token in order (BY_MASS false), or the first at which the
// running weight reaches `want`. Only tokens at or above `floor` and in bins up to `last_bin`
// count. 0: the border lies among weights of zero.
template <bool BY_MASS, typename R>
__device__ u64 find_border(const cg::cluster_group& cluster, SampleShared& sh, const R& row, const Weighing& weigh, u64 want, u64 floor, int last_bin) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  SampleShared& lead = *cluster.map_shared_rank(&sh, 0);
  const bool is_lead = cluster.block_rank() == 0;
  uint32_t* const count = reinterpret_cast<uint32_t*>(sh.hist);
  u64 prefix = 0, prefix_mask = 0;
  int only_bin = -1;
  for (int shift = 64;;) {  // first the bins, then 12 bits of the order at a time from the top
    for (int i = tid; i < BINS; i += SAMPLE_THREADS) sh.hist[i] = 0;
    if (is_lead && tid == 0) sh.listed = 0;
    cluster.sync();  // the first CTA's histogram is empty before any other adds to it
    row.each([&](float x, int i) {
      const int b = weigh.bin_of(x);
      if (b > last_bin || (only_bin >= 0 && b != only_bin)) return;
      const u64 o = order_of(x, i);
      if (o < floor || (o & prefix_mask) != prefix) return;
      const int at = shift == 64 ? b : BINS - 1 - static_cast<int>((o >> shift) & (BINS - 1));
      if (BY_MASS) atomicAdd(&sh.hist[at], weigh.of(x));
      else atomicAdd(&count[at], 1u);
    });
    __syncthreads();
    if (!is_lead) {
      uint32_t* const lead_count = reinterpret_cast<uint32_t*>(lead.hist);
      for (int i = tid; i < BINS; i += SAMPLE_THREADS) {
        if (BY_MASS) { if (sh.hist[i]) atomicAdd(&lead.hist[i], sh.hist[i]); }
        else { if (count[i]) atomicAdd(&lead_count[i], count[i]); }
      }
    }
    cluster.sync();
    if (is_lead) {
      constexpr int RUN = BINS / SAMPLE_THREADS;
      u64 mine = 0;
#pragma unroll
      for (int i = 0; i < RUN; ++i) mine += BY_MASS ? sh.hist[tid * RUN + i] : count[tid * RUN + i];
      u64 incl = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
      }
      if (lane == 31) sh.red[warp] = incl;
      if (tid == 0) sh.found = -1;
      __syncthreads();
      u64 sum = incl - mine;
      for (int w = 0; w < warp; ++w) sum += sh.red[w];
      if (sum < want && want <= sum + mine) {
        int b = tid * RUN;
        for (;; ++b) {
          const u64 here = BY_MASS ? sh.hist[b] : count[b];
          if (want <= sum + here) break;
          sum += here;
        }
        sh.found = b;
        sh.above = sum;
      }
      __syncthreads();
      if (tid < static_cast<int>(cluster.num_blocks())) {
        SampleShared& other = *cluster.map_shared_rank(&sh, tid);
        other.bin = sh.found;
        if (tid) other.above = sh.above;
      }
    }
    cluster.sync();
    const int bin = sh.bin;
    if (bin < 0) return 0;
    want -= sh.above;
    if (shift == 64) only_bin = bin;
    else {
      prefix |= static_cast<u64>(BINS - 1 - bin) << shift;
      prefix_mask |= static_cast<u64>(BINS - 1) << shift;
    }
    // the bin's tokens, ranked by the first CTA if they are few enough
    row.each([&](float x, int i) {
      if (weigh.bin_of(x) != only_bin) return;
      const u64 o = order_of(x, i);
      if (o < floor || (o & prefix_mask) != prefix) return;
      const int at = atomicAdd(&lead.listed, 1);
      if (at < LIST) {
        lead.list[at] = o;
        if (BY_MASS) lead.mass[at] = weigh.of(x);
      }
    });
    cluster.sync();
    const int listed = lead.listed;
    if (listed <= LIST) {
      if (is_lead) {
        if (tid < listed) {
          const u64 o = sh.list[tid];
          u64 before = 0;
          for (int i = 0; i < listed; ++i)
            if (sh.list[i] > o) before += BY_MASS ? sh.mass[i] : 1;
          if (before < want && want <= before + (BY_MASS ? sh.mass[tid] : 1)) sh.border = o;
        }
        __syncthreads();
        if (tid > 0 && tid < static_cast<int>(cluster.num_blocks())) cluster.map_shared_rank(&sh, tid)->border = sh.border;
      }
      cluster.sync();
      return sh.border;
    }
    shift = shift == 64 ? 40 : shift > 12 ? shift - 12 : 0;  // 52 bits: 40, 28, 16, 4, 0
    cluster.sync();  // everyone has read `listed` before it is cleared
  }
}

template <bool HELD>
__global__ void __launch_bounds__(SAMPLE_THREADS, 2) sample_kernel(const SampleParams p) {
  __shared__ SampleShared sh;
  extern __shared__ float held[];
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();  // waited for below: nobody writes to a CTA that has not started
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int r = blockIdx.x / ctas;
  Row<HELD> row;
  row.held = held;
  row.logits = p.logits;
  row.dtype = p.dtype;
  row.base = r * p.row_stride;
  row.vocab = p.vocab;
  row.steps = p.items;
  row.offset = warp * 32 * p.items + lane;  // a warp owns a run: index order is CTA, warp, step, lane
  row.first = rank * SAMPLE_THREADS * p.items + row.offset;
  if (HELD) {
#pragma unroll 16
    for (int j = 0; j < p.items; ++j) {
      const int i = row.first + j * 32;
      held[row.offset + j * 32] = i < p.vocab ? load_as_f32(p.logits, p.dtype, row.base + i) : 0.f;  // only this lane reads it back
    }
  }
  if (tid < TABLE) sh.table[tid] = exp2(WEIGHT_BITS + static_cast<double>(tid) / TABLE);
  auto finish = [&](int64_t token, float lp) {
    if (p.tok64) static_cast<int64_t*>(p.tokens)[r * p.stok] = token;
    else static_cast<int32_t*>(p.tokens)[r * p.stok] = static_cast<int32_t>(token);
    if (p.logprobs) p.logprobs[r * p.slp] = lp;
  };
  // the first in order
  u64 best = 0;
  row.each([&](float x, int i) {
    const u64 o = order_of(x, i);
    if (o > best) best = o;
  });
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const u64 o = __shfl_xor_sync(0xffffffffu, best, d);
    if (o > best) best = o;
  }
  if (lane == 0) sh.red[warp] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) best = sh.red[w] > best ? sh.red[w] : best;
  cluster.barrier_wait();
  exchange(cluster, sh, 0, best);
  for (int c = 0; c < ctas; ++c) best = sh.from[0][c] > best ? sh.from[0][c] : best;
  const float top = logit_of(best);
  const float temperature = p.temperature ? p.temperature[r * p.st] : 1.f;
  const float top_p = p.top_p ? p.top_p[r * p.sp] : 1.f;
  const float min_p = p.min_p ? p.min_p[r * p.sm] : 0.f;
  const int64_t k = p.top_k ? (p.k64 ? static_cast<const int64_t*>(p.top_k)[r * p.sk] : static_cast<const int32_t*>(p.top_k)[r * p.sk]) : 0;
  if (top == -INFINITY || !(temperature > 0.f) || k == 1 || top_p <= 0.f) {  // the whole cluster leaves; nobody's memory is asked for any more
    if (rank == 0 && tid == 0) {
      if (top == -INFINITY) finish(-1, -INFINITY);
      else finish(index_of(best), 0.f);
    }
    return;
  }
  Weighing weigh;
  weigh.top = top;
  weigh.top64 = static_cast<double>(top);
  weigh.scale = TABLE * 1.4426950408889634073599 / static_cast<double>(temperature);
  weigh.bin_scale = 2.f * BINS_PER_OCTAVE * 1.44269504f / temperature;
  weigh.table = sh.table;

  u64 border = 0;  // kept: this place in the order and before
  if (k > 0 && k < p.vocab) border = find_border<false>(cluster, sh, row, weigh, static_cast<u64>(k), 0, BINS - 2);
  if (top_p < 1.f) {
    u64 sum = 0;
    row.each([&](float x, int i) {
      if (order_of(x, i) >= border) sum += weigh.of(x);
    });
    sum = block_total(sum, sh.red);
    exchange(cluster, sh, 1, sum);
    sum = 0;
    for (int c = 0; c < ctas; ++c) sum += sh.from[1][c];
    // a whole number reaches p * sum when it reaches the next whole number; p < 1 keeps that within the sum
    const u64 need = __double2ull_ru(static_cast<double>(top_p) * static_cast<double>(sum));
    // Tokens lighter than (sum - need) / vocab are beyond the border: all together they do not make
    // up what may be left out. One bin of margin covers the bins' f32 arithmetic.
    const u64 light = (sum - need) / static_cast<u64>(p.vocab);
    int last_bin = BINS - 2;
    if (light > 0) last_bin = min(last_bin, static_cast<int>((WEIGHT_BITS - log2f(static_cast<float>(light))) * BINS_PER_OCTAVE) + 2);
    border = find_border<true>(cluster, sh, row, weigh, need, border, last_bin);
  }
  const u64 least = min_p > 0.f ? __double2ull_ru(fmin(static_cast<double>(min_p), 1.0) * static_cast<double>(WEIGHT_ONE)) : 0;
  auto kept_weight = [&](float x, int i) -> u64 {
    if (order_of(x, i) < border) return 0;
    const u64 w = weigh.of(x);
    return w >= least ? w : 0;  // the largest weighs 2^42: it always stays
  };
  u64 mine = 0;
  row.each([&](float x, int i) { mine += kept_weight(x, i); });
  mine = warp_total(mine);
  __syncthreads();
  if (lane == 0) sh.red[warp] = mine;
  __syncthreads();
  u64 here = 0, before = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += sh.red[w];
    here += sh.red[w];
  }
  exchange(cluster, sh, 2, here);
  u64 total = 0;
  for (int c = 0; c < ctas; ++c) {
    if (c < rank) before += sh.from[2][c];
    total += sh.from[2][c];
  }
  // the first index whose running sum is above u * total; a number at or beyond 1 takes the last
  const float u = p.uniform[r * p.su];
  const u64 target = !(u > 0.f) ? 0 : u >= 1.f ? total - 1 : __double2ull_rd(static_cast<double>(u) * static_cast<double>(total));
  if (before <= target && before + mine > target) {  // one warp of the cluster
    for (int j = 0; j < p.items; ++j) {
      const int i = row.first + j * 32;
      const u64 w = i < p.vocab ? kept_weight(load_as_f32(p.logits, p.dtype, row.base + i), i) : 0;
      u64 incl = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + incl > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) finish(i, static_cast<float>(log(static_cast<double>(w) / static_cast<double>(total))));
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
}

// Values per thread that fit a CTA's shared memory beside its tables; with 32 or fewer two CTAs
// share an SM, and one loads while the other computes.
constexpr int MOST_HELD = 64;

bool vector_of(const lh_memref_t* m, int64_t n) { return m->rank == 1 && m->shape[0] == n; }

}  // namespace
}  // namespace lh

using namespace lh;

extern "C" int lh_b200_sample(lh_ctx_t* ctx, const lh_memref_t* tokens, const lh_memref_t* logprobs, const lh_memref_t* logits, const lh_memref_t* uniform,
                              const lh_memref_t* temperature, const lh_memref_t* top_k, const lh_memref_t* top_p, const lh_memref_t* min_p) {
  if (!ctx) return LH_ERR_INVALID;
  if (!tokens || !logits || !uniform) return set_error(ctx, LH_ERR_INVALID, "sample: tokens, logits and uniform are required");
  if (logits->rank != 2) return set_error(ctx, LH_ERR_INVALID, "sample: logits are (rows, vocabulary)");
  const int64_t n = logits->shape[0], v = logits->shape[1];
  if (n < 0 || n > 0x7fffffffll || v < 1) return set_error(ctx, LH_ERR_INVALID, "sample: logits of %lld x %lld", (long long)n, (long long)v);
  if (v > MAX_VOCAB) return set_error(ctx, LH_ERR_UNSUPPORTED, "sample: a vocabulary of %lld is above %lld", (long long)v, (long long)MAX_VOCAB);
  if (logits->dtype != LH_F32 && logits->dtype != LH_BF16 && logits->dtype != LH_F16) return set_error(ctx, LH_ERR_UNSUPPORTED, "sample: f32, bf16 or f16 logits");
  if (v > 1 && logits->strides[1] != 1) return set_error(ctx, LH_ERR_UNSUPPORTED, "sample: a row of logits must have unit stride");
  for (const lh_memref_t* m : {tokens, logprobs, uniform, temperature, top_k, top_p, min_p})
    if (m && !vector_of(m, n)) return set_error(ctx, LH_ERR_INVALID, "sample: tokens, logprobs, uniform and the settings have one entry per row");
  for (const lh_memref_t* m : {logprobs, uniform, temperature, top_p, min_p})
    if (m && m->dtype != LH_F32) return set_error(ctx, LH_ERR_INVALID, "sample: logprobs, uniform, temperature, top_p and min_p are f32");
  for (const lh_memref_t* m : {tokens, top_k})
    if (m && m->dtype != LH_I32 && m->dtype != LH_I64) return set_error(ctx, LH_ERR_INVALID, "sample: tokens and top_k are i32 or i64");
  for (const lh_memref_t* m : {tokens, logprobs})
    if (m && n > 1 && m->strides[0] == 0) return set_error(ctx, LH_ERR_INVALID, "sample: a written operand overlaps itself (zero stride)");
  if (n == 0) return LH_OK;
  SampleParams p;
  memset(&p, 0, sizeof(p));
  p.logits = data_ptr(logits); p.row_stride = logits->strides[0]; p.dtype = logits->dtype;
  p.rows = static_cast<int>(n); p.vocab = static_cast<int>(v);
  auto f32 = [](const lh_memref_t* m, int64_t& stride) -> float* {
    if (!m) return nullptr;
    stride = m->strides[0];
    return reinterpret_cast<float*>(data_ptr(m));
  };
  p.uniform = f32(uniform, p.su);
  p.temperature = f32(temperature, p.st);
  p.top_p = f32(top_p, p.sp);
  p.min_p = f32(min_p, p.sm);
  p.logprobs = f32(logprobs, p.slp);
  if (top_k) { p.top_k = data_ptr(top_k); p.sk = top_k->strides[0]; p.k64 = top_k->dtype == LH_I64; }
  p.tokens = data_ptr(tokens); p.stok = tokens->strides[0]; p.tok64 = tokens->dtype == LH_I64;
  // Small rows take one CTA. Larger ones take up to eight, four values per thread and more: what a
  // row costs is mostly latency (barriers, histograms), so the wider it is spread the sooner it
  // ends, and eight is the largest cluster that every launch may have.
  int ctas = 1;
  while (ctas < MAX_CLUSTER && v > static_cast<int64_t>(ctas) * SAMPLE_THREADS * 4) ctas *= 2;
  p.items = static_cast<int>((v + static_cast<int64_t>(ctas) * SAMPLE_THREADS - 1) / (static_cast<int64_t>(ctas) * SAMPLE_THREADS));
  if (n > 0x7fffffffll / ctas) return set_error(ctx, LH_ERR_UNSUPPORTED, "sample: %lld rows are too many for one call", (long long)n);
  DeviceScope scope(ctx->device);
  const bool held = p.items <= MOST_HELD;
  const size_t smem = held ? static_cast<size_t>(p.items) * SAMPLE_THREADS * sizeof(float) : 0;
  if (held) LH_CUDA_CHECK(ctx, cudaFuncSetAttribute(sample_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_HELD * SAMPLE_THREADS * static_cast<int>(sizeof(float))));
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(n * ctas));
  cfg.blockDim = dim3(SAMPLE_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LH_CUDA_CHECK(ctx, cudaLaunchKernelEx(&cfg, held ? sample_kernel<true> : sample_kernel<false>, p));
  LH_CHECK_LAUNCH(ctx, "sample_kernel");
  return LH_OK;
}
