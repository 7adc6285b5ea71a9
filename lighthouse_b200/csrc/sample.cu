// Sampling a token per row of logits. Entry point lh_b200_sample.
//
// Weights are whole numbers: w = round(2^42 exp((x - max) / T)), formed in f64. Sums of them are
// exact, so they come out the same in whatever order threads and CTAs add them, and a
// drawn token does not depend on how the row was cut up. In f32 the running sum of 10^5 weights
// is off by 1e-7 of the total, and as many borders between tokens lie in it: one row in some
// hundreds would get another token than the definition gives.
#include "common.cuh"
#include "epilogue.cuh"

namespace lh {
namespace {

struct SampleParams {
  const void* logits; int64_t row_stride; int dtype;
  int rows, vocab;
  const float* uniform; int64_t su;
  const float* temperature; int64_t st;
  const void* top_k; int64_t sk; int k64;
  const float* top_p; int64_t sp;
  const float* min_p; int64_t sm;
  void* tokens; int64_t stok; int tok64;
  float* logprobs; int64_t slp;
};

constexpr double WEIGHT_ONE = 4398046511104.0;  // 2^42: the largest weight
constexpr int WEIGHT_BITS = 42;
constexpr int64_t MAX_VOCAB = int64_t(1) << 20;  // 2^20 weights of 2^42 stay within 63 bits
constexpr int SAMPLE_THREADS = 1024;
constexpr int WARPS = SAMPLE_THREADS / 32;

// Values in an order that whole numbers keep; NaN ranks with -inf, -0 with +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x == x)) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }

struct Weighing {
  double top, scale;  // row maximum, log2(e) / T
  // log2 of the weight: 0 for the maximum
  __device__ __forceinline__ double log2_of(float x) const {
    const double d = static_cast<double>(x);
    return d == top ? 0.0 : (d - top) * scale;
  }
  __device__ __forceinline__ unsigned long long of(float x) const {
    const double t = log2_of(x);
    if (!(t > -(WEIGHT_BITS + 1.0)) || x == -INFINITY) return 0;  // also NaN: (-inf) * 0
    return static_cast<unsigned long long>(__double2ll_rn(exp2(t) * WEIGHT_ONE));
  }
};

template <typename V>
__device__ __forceinline__ V warp_total(V v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

__device__ unsigned long long block_total(unsigned long long v, unsigned long long* red) {
  v = warp_total(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < WARPS; ++w) v += red[w];
  return v;
}

// One CTA per row; each warp owns a run of the row, so that index order is warp order.
__global__ void __launch_bounds__(SAMPLE_THREADS) sample_kernel(const SampleParams p) {
  __shared__ unsigned long long red[WARPS];
  __shared__ unsigned long long mass[256];
  __shared__ int count[256];
  __shared__ unsigned long long sh_mass;
  __shared__ int sh_digit, sh_count, sh_index;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x;
  const int64_t base = row * p.row_stride;
  const int run = ((p.vocab + WARPS - 1) / WARPS + 31) / 32 * 32;
  const int w0 = min(warp * run, p.vocab), w1 = min(w0 + run, p.vocab);
  auto value = [&](int i) { return load_as_f32(p.logits, p.dtype, base + i); };
  auto finish = [&](int64_t token, float lp) {
    if (tid == 0) {
      if (p.tok64) static_cast<int64_t*>(p.tokens)[row * p.stok] = token;
      else static_cast<int32_t*>(p.tokens)[row * p.stok] = static_cast<int32_t>(token);
      if (p.logprobs) p.logprobs[row * p.slp] = lp;
    }
  };
  // the largest key, and the first index that has it
  unsigned long long best = 0;
  for (int i = w0 + lane; i < w1; i += 32) {
    const unsigned long long k = (static_cast<unsigned long long>(key_of(value(i))) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
    if (k > best) best = k;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, best, d);
    if (o > best) best = o;
  }
  if (lane == 0) red[warp] = best;
  __syncthreads();
  best = 0;
  for (int w = 0; w < WARPS; ++w) best = red[w] > best ? red[w] : best;
  const uint32_t key_max = static_cast<uint32_t>(best >> 32);
  const int first_max = static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
  const float top = value_of(key_max);
  if (top == -INFINITY) return finish(-1, -INFINITY);
  const float temperature = p.temperature ? p.temperature[row * p.st] : 1.f;
  const float top_p = p.top_p ? p.top_p[row * p.sp] : 1.f;
  const float min_p = p.min_p ? p.min_p[row * p.sm] : 0.f;
  int64_t k = p.top_k ? (p.k64 ? static_cast<const int64_t*>(p.top_k)[row * p.sk] : static_cast<const int32_t*>(p.top_k)[row * p.sk]) : 0;
  if (!(temperature > 0.f) || k == 1 || top_p <= 0.f) return finish(first_max, 0.f);
  Weighing weigh;
  weigh.top = static_cast<double>(top);
  weigh.scale = 1.4426950408889634073599 / static_cast<double>(temperature);

  // Kept so far: keys above `key`, and the first `ties` of those equal to it.
  uint32_t key = 0;
  int64_t ties = p.vocab;
  if (k > 0 && k < p.vocab) {
    // the k-th largest key, eight bits at a time
    int64_t left = k;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) count[tid] = 0;
      __syncthreads();
      const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for (int i = w0 + lane; i < w1; i += 32) {
        const uint32_t q = key_of(value(i));
        if ((q & mask) == key) atomicAdd(&count[(q >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255;
        int64_t rest = left;
        while (d > 0 && count[d] < rest) rest -= count[d--];
        sh_digit = d;
        sh_count = static_cast<int>(rest);
      }
      __syncthreads();
      key |= static_cast<uint32_t>(sh_digit) << shift;
      left = sh_count;
      __syncthreads();
    }
    ties = left;
  }
  if (top_p < 1.f) {
    // total weight of what is left, then the key at which the running sum, taken from the largest
    // weight down, reaches its share
    unsigned long long sum = 0;
    for (int i = w0 + lane; i < w1; i += 32) {
      const float x = value(i);
      if (key_of(x) > key) sum += weigh.of(x);
    }
    sum = block_total(sum, red);
    if (key) sum += static_cast<unsigned long long>(ties) * weigh.of(value_of(key));
    // a whole number reaches p * sum when it reaches the next whole number
    const unsigned long long need = __double2ull_ru(static_cast<double>(top_p) * static_cast<double>(sum));
    unsigned long long above = 0;
    uint32_t at = 0;
    int64_t equal = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) { mass[tid] = 0; count[tid] = 0; }
      __syncthreads();
      const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for (int i = w0 + lane; i < w1; i += 32) {
        const float x = value(i);
        const uint32_t q = key_of(x);
        if ((q & mask) == at && q >= key) {
          atomicAdd(&mass[(q >> shift) & 255], weigh.of(x));
          atomicAdd(&count[(q >> shift) & 255], 1);
        }
      }
      __syncthreads();
      if (tid == 0) {
        // p < 1 keeps `need` within the sum, and ties of `key` beyond the first `ties`, which are
        // not in the sum, lie in the last bin that holds anything: the walk ends in a bin
        unsigned long long run_sum = above;
        int d = 255;
        while (d > 0 && run_sum + mass[d] < need) run_sum += mass[d--];
        sh_digit = d;
        sh_mass = run_sum;
        sh_count = count[d];
      }
      __syncthreads();
      at |= static_cast<uint32_t>(sh_digit) << shift;
      above = sh_mass;
      equal = sh_count;
      __syncthreads();
    }
    if (at > key || !key) ties = equal;  // all of them, before the share is counted
    key = at;
    const unsigned long long each = weigh.of(value_of(key));
    // each > 0: `above` alone falls short of `need`
    const int64_t want = static_cast<int64_t>((need - above + each - 1) / each);
    if (want < ties) ties = want;
  }
  // the index of the last tie that is kept
  int last_tie = p.vocab;
  if (key) {
    int here = 0;
    for (int i = w0 + lane; i < w1; i += 32) here += key_of(value(i)) == key;
    here = warp_total(here);
    __syncthreads();
    if (lane == 0) red[warp] = static_cast<unsigned long long>(here);
    if (tid == 0) sh_index = p.vocab;
    __syncthreads();
    int64_t before = 0;
    for (int w = 0; w < warp; ++w) before += static_cast<int64_t>(red[w]);
    if (before < ties && before + here >= ties) {
      int64_t seen = before;
      for (int i0 = w0; i0 < w1; i0 += 32) {
        const int i = i0 + lane;
        const unsigned hit = __ballot_sync(0xffffffffu, i < w1 && key_of(value(i)) == key);
        if (seen + __popc(hit) >= ties) {
          const int nth = static_cast<int>(ties - seen);  // the nth set bit
          if ((hit >> lane & 1) && __popc(hit & ((2u << lane) - 1)) == nth) sh_index = i;
          break;
        }
        seen += __popc(hit);
      }
    }
    __syncthreads();
    last_tie = sh_index;
  }
  const double floor2 = min_p > 0.f ? log2(static_cast<double>(min_p)) : -INFINITY;
  auto kept_weight = [&](int i) -> unsigned long long {
    const float x = value(i);
    const uint32_t q = key_of(x);
    if (q < key || (q == key && i > last_tie)) return 0;
    if (!(x == x)) return 0;
    if (q != key_max && !(weigh.log2_of(x) >= floor2)) return 0;
    return weigh.of(x);
  };
  unsigned long long mine = 0;
  for (int i = w0 + lane; i < w1; i += 32) mine += kept_weight(i);
  mine = warp_total(mine);
  __syncthreads();
  if (lane == 0) red[warp] = mine;
  if (tid == 0) sh_index = -1;
  __syncthreads();
  unsigned long long total = 0, before = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += red[w];
    total += red[w];
  }
  // the first index whose running sum is above u * total; a number at or beyond 1 takes the last
  const float u = p.uniform[row * p.su];
  const unsigned long long target = !(u > 0.f) ? 0 : u >= 1.f ? total - 1 : __double2ull_rd(static_cast<double>(u) * static_cast<double>(total));
  if (before <= target && before + mine > target) {
    unsigned long long sum = before;
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const int i = i0 + lane;
      const unsigned long long w = i < w1 ? kept_weight(i) : 0;
      unsigned long long incl = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned long long up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, sum + incl > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          sh_index = i;
          sh_mass = w;
        }
        break;
      }
      sum += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  __syncthreads();
  finish(sh_index, static_cast<float>(log(static_cast<double>(sh_mass) / static_cast<double>(total))));
}

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
  DeviceScope scope(ctx->device);
  sample_kernel<<<static_cast<unsigned>(n), SAMPLE_THREADS, 0, ctx->stream>>>(p);
  LH_CHECK_LAUNCH(ctx, "sample_kernel");
  return LH_OK;
}
