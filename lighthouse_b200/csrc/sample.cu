// Sampling a token per row of logits. Entry point lh_b200_sample.
//
// Weights are whole numbers: w = floor(2^42 exp((x - max) / T)), formed in f64. Sums of them are
// exact, so they come out the same in whatever order threads and CTAs add them, and a
// drawn token does not depend on how the row was cut up. In f32 the running sum of 10^5 weights
// is off by 1e-7 of the total, and as many borders between tokens lie in it: one row in some
// hundreds would get another token than the definition gives.
//
// A row belongs to a cluster of CTAs, which talk through distributed shared memory; the first
// of them (the lead) adds up and decides. What top-k and top-p keep is always "the first so many
// in the order of falling logits, equal ones by rising index", so each is one border in that
// order, found in two steps: a histogram over log2 of the weight (4096 bins of 1/93 octave) says
// which bins the border can lie in, and their few dozen tokens are collected and ranked against
// each other by the lead. For top-k the bins count tokens; for top-p they add up weights in units of
// 2^-13 or 2^-11, and the exact sums outside the candidate bins, formed while the candidates are collected,
// both complete the decision and show that the bins were the right ones. Candidates too many to
// rank (rows of equal logits) are narrowed by digits of the order itself first. What top-k leaves
// is usually few: then the lead is sent all of it and does the rest by itself.
//
// The row is read from global memory by every pass (three for top-p), 16 bytes at a time, after
// the first pass from L1 and L2. 256 rows of 131071 f32 logits with top-p take 175 us; reading them once
// would take 20, and 64 bf16 rows of mixed settings 63 us (2.6). What bounds a full batch is the
// instructions and their latency, not the memory: issue slots are taken for 53 % of the time with the 32
// warps an SM has room for, the f64 pipe for 13 %. The exact pass takes 55 clocks of a scheduler for a
// warp's 32 weights (ten f64 operations each, about as many others), the histogram 25 (it goes by an f32
// coordinate), the maximum 20, and a fifth of the time goes to the cluster's barriers around them. So a weight
// is formed once per token. Running sums are kept in f64 with 2^52 added: adding with rounding down
// then drops each weight's fraction, whatever the sum so far. One row of 50304 takes 17 us: steps
// across the cluster, one after the other.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace lh {
namespace {

struct SampleParams {
  const void* logits; int64_t row_stride;
  int vocab;
  int steps;  // 16-byte groups per thread: a warp has a run of 32 * steps groups of the row, a CTA WARPS runs
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
constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int CTAS_PER_SM = 2;  // 64 registers: the weights' f64 chains interleave (three CTAs at 40 registers spill, and measured the same)
constexpr int MAX_CLUSTER = 8;
constexpr int MAX_RUNS = MAX_CLUSTER * WARPS;
constexpr int BINS = 4096;
constexpr int WIDE = 1 << 18;  // rows up to this add up weights to 2^-13, wider ones to 2^-11
constexpr float BINS_PER_OCTAVE = 93.f;  // the last bin starts 44 octaves below the maximum: weights of zero
constexpr int DIGIT_BITS = 11;
constexpr int DIGITS = 1 << DIGIT_BITS;
constexpr int LIST = 1024;
constexpr int TABLE = 64;
constexpr int COPIES = 16;  // of the table: the half of a warp that a 64-bit load serves at a time finds a bank for each lane

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

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

// A running sum of whole weights, at most 2^10 of them.
struct Tally {
  double sum = 4503599627370496.0;  // 2^52: its last bit counts ones
  __device__ __forceinline__ Tally& add(double w) {
    sum = __dadd_rd(sum, w);
    return *this;
  }
  __device__ __forceinline__ u64 value() const { return static_cast<u64>(__double_as_longlong(sum)) & ((1ull << 52) - 1); }
};

struct Weighing {
  float top, half_top;
  float bin_scale;       // bins per two units of logit
  float lowest;          // what is not above it (NaN is not) weighs nothing
  double top64, scale;   // row maximum; 64 log2(e) / T
  const double* table;   // 2^(42 + i / 64), this lane's copy

  // Distance from the maximum in bins. Falls with x; 0 for the maximum, BINS - 1 for NaN, -inf and
  // whatever weighs nothing. (Halves: the difference of two finite logits stays finite.)
  __device__ __forceinline__ float place_of(float x) const { return fminf(fmaf(x, -0.5f, half_top) * bin_scale, static_cast<float>(BINS - 1)); }
  // Rounding towards zero by adding 2^23 keeps the conversion off the slow units.
  __device__ __forceinline__ int bin_of(float x) const { return __float_as_int(__fadd_rd(place_of(x), 8388608.f)) & (BINS - 1); }

  // 2^42 times the weight, not yet a whole number, of a logit above `lowest`.
  // 2^t = 2^(j / 64) (1 + (e^(f ln2 / 64) - 1)), 64 t = j + f, |f| <= 1/2: the series' fifth term
  // and on are below 2^-44.
  __device__ __forceinline__ double of(float x) const {
    const double d = static_cast<double>(x) - top64;
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the nearest whole number
    const double z = fma(d, scale, magic);
    const int j = __double2loint(z);
    const double f = fma(d, scale, magic - z);
    constexpr double a1 = 0.69314718055994530942 / TABLE, a2 = a1 * a1 / 2, a3 = a2 * a1 / 3, a4 = a3 * a1 / 4;
    const double s = f * fma(f, fma(f, fma(f, a4, a3), a2), a1);
    const int low = j & (TABLE - 1);
    const double base = table[low * COPIES];
    const double scaled = __hiloint2double(__double2hiint(base) + (j - low) * ((1 << 20) / TABLE), __double2loint(base));
    return fma(scaled, s, scaled);
  }
  __device__ __forceinline__ bool counts(float x) const { return x > lowest; }
  __device__ __forceinline__ u64 whole(float x) const {
    const u64 w = Tally().add(of(x)).value();  // (whatever it is at logits that do not count)
    return w & (counts(x) ? ~0ull : 0ull);
  }
};

template <typename V>
__device__ __forceinline__ V warp_total(V v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
template <typename V>
__device__ __forceinline__ V warp_inclusive(V v) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) >= d) v += up;
  }
  return v;
}

enum Verdict : int { FOUND, NOTHING, TOO_MANY, WRONG_BINS, ALL_LISTED };

// What the lead tells every CTA.
struct Answer {
  u64 border;          // kept: this place in the order and before
  u64 want;            // of the candidates' count or weight, up to the border
  u64 prefix;          // digits of the border's place known so far
  u64 total, residual; // kept weight; how far into the owner's run the draw lies
  float from, to;      // candidates' logits are in (to, from]
  int verdict;
  int owner;           // the run that the draw lies in
};
static_assert(sizeof(Answer) % sizeof(u64) == 0, "copied in words");

struct Shared {
  double table[TABLE * COPIES];
  u64 digits[DIGITS];      // sums of a digit; or, as 32-bit words, of the bins
  // The CTA's candidates, and in the lead everybody's (`mass` by place in the list). Between uses of
  // the list the lead keeps the cluster's sums of bins or digits here.
  u64 list[LIST], mass[LIST];
  u64 kept[MAX_RUNS], middle[MAX_RUNS], all[MAX_RUNS];  // lead: weights before the candidates, of them and of everything, per run
  u64 red[WARPS];
  Answer answer;
  float tops[MAX_CLUSTER];
  int firsts[MAX_CLUSTER];
  int listed, counts[MAX_CLUSTER];
  int lo, hi;
};
static_assert(sizeof(u64) * DIGITS == sizeof(uint32_t) * BINS && DIGITS == 2 * LIST, "bins and digits share their memory, sums of either fit the list's");

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
// Sum of the threads before this one; `all` the block's.
template <typename V>
__device__ __forceinline__ V block_before(V v, V* red, V& all) {
  const V incl = warp_inclusive(v);
  const int warp = threadIdx.x >> 5;
  __syncthreads();
  if ((threadIdx.x & 31) == 31) red[warp] = incl;
  __syncthreads();
  V before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += red[w];
    all += red[w];
  }
  return before + incl - v;
}

// The first index whose running sum is above u * total is drawn; a number at or beyond 1 takes the last.
__device__ __forceinline__ u64 target_of(float u, u64 total) {
  return !(u > 0.f) ? 0 : u >= 1.f ? total - 1 : __double2ull_rd(static_cast<double>(u) * static_cast<double>(total));
}
// A whole number reaches p * sum when it reaches the next whole number; p < 1 keeps that within the sum.
__device__ __forceinline__ u64 share_of(float p, u64 sum) { return __double2ull_ru(static_cast<double>(p) * static_cast<double>(sum)); }
__device__ __forceinline__ float log_share(u64 w, u64 total) { return static_cast<float>(log(static_cast<double>(w) / static_cast<double>(total))); }
__device__ __forceinline__ void finish(const SampleParams& p, int r, int64_t token, float logprob) {
  if (p.tok64) static_cast<int64_t*>(p.tokens)[r * p.stok] = token;
  else static_cast<int32_t*>(p.tokens)[r * p.stok] = static_cast<int32_t>(token);
  if (p.logprobs) p.logprobs[r * p.slp] = logprob;
}

template <typename T>
struct Sampler {
  static constexpr int VEC = 16 / sizeof(T);
  static constexpr int BATCH = sizeof(T) == 4 ? 4 : 2;  // groups in flight per thread: sixteen values
  cg::cluster_group cluster;
  Shared& sh;
  Shared& lead;
  const T* row;
  int run, ctas, rank, vocab, steps;
  int head, tail;       // where the row's whole 16-byte groups begin and end; the first run has what is before, the last what is behind
  int begin, end;       // this thread's first group, and where the groups of its run end
  Weighing weigh;

  __device__ __forceinline__ void cut() {
    const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
    head = min(vocab, skew ? VEC - skew : 0);
    begin = run * 32 * steps + (threadIdx.x & 31);
    end = min((run + 1) * 32 * steps, (vocab - head) / VEC);
    tail = head + (vocab - head) / VEC * VEC;
  }
  __device__ __forceinline__ int run_length() const { return 32 * VEC * steps; }
  __device__ __forceinline__ int runs() const { return ctas * WARPS; }
  __device__ __forceinline__ int run_of(int i) const { return i < head ? 0 : i >= tail ? runs() - 1 : (i - head) / run_length(); }
  // f(value, index). Sixteen values are unrolled: their f64 chains interleave. (A rolled loop that loads
  // ahead, four values a turn, took 1.3 times as long.)
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const T* const origin = row + head;
    int g = begin;
#pragma unroll 1
    for (; g + 32 * (BATCH - 1) < end; g += 32 * BATCH) {
      uint4 raw[BATCH];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) raw[b] = *reinterpret_cast<const uint4*>(origin + (g + b * 32) * VEC);
#pragma unroll
      for (int b = 0; b < BATCH; ++b)
#pragma unroll
        for (int v = 0; v < VEC; ++v) f(as_f32(reinterpret_cast<const T*>(&raw[b])[v]), head + (g + b * 32) * VEC + v);
    }
#pragma unroll 1
    for (; g < end; g += 32) {
      const uint4 raw = *reinterpret_cast<const uint4*>(origin + g * VEC);
#pragma unroll
      for (int v = 0; v < VEC; ++v) f(as_f32(reinterpret_cast<const T*>(&raw)[v]), head + g * VEC + v);
    }
    // the odd ends, fewer than VEC values each: one per lane
    const int lane = threadIdx.x & 31;
    const int i = run == 0 && lane < head ? lane : run == runs() - 1 && lane >= 16 ? tail + lane - 16 : vocab;
    if (i < vocab) f(as_f32(row[i]), i);
  }
  __device__ __forceinline__ bool is_lead() const { return rank == 0; }

  // The lead's answer reaches every CTA. Ends with a barrier.
  __device__ __forceinline__ void tell() {
    if (is_lead()) {
      __syncthreads();
      constexpr int WORDS = sizeof(Answer) / sizeof(u64);
      for (int i = threadIdx.x; i < WORDS * (ctas - 1); i += THREADS)
        reinterpret_cast<u64*>(&cluster.map_shared_rank(&sh, 1 + i / WORDS)->answer)[i % WORDS] = reinterpret_cast<const u64*>(&sh.answer)[i % WORDS];
    }
    cluster.sync();
  }

  // Adds up the CTAs' bins (or digits) for the lead: every CTA sums a part of them over the cluster.
  // (One read of everything by the lead, or everybody adding to the lead's, queues at one SM.)
  template <typename V>
  __device__ V* sum_up(V* mine, int n) {
    V* const sums = reinterpret_cast<V*>(sh.list);
    cluster.sync();
    V* const to = cluster.map_shared_rank(sums, 0);
    const int part = n / ctas;
    for (int i = rank * part + threadIdx.x; i < (rank + 1) * part; i += THREADS) {
      V v[MAX_CLUSTER], sum = 0;
#pragma unroll
      for (int c = 0; c < MAX_CLUSTER; ++c) v[c] = c < ctas ? cluster.map_shared_rank(mine, c)[i] : 0;
#pragma unroll
      for (int c = 0; c < MAX_CLUSTER; ++c) sum += v[c];
      to[i] = sum;
    }
    cluster.sync();
    clear_bins();
    return sums;
  }

  __device__ __forceinline__ void clear_bins() {
    for (int i = threadIdx.x; i < DIGITS; i += THREADS) sh.digits[i] = 0;
  }

  // The largest logit whose bin is at least b (b > 0): what is above it is in an earlier bin. One warp
  // searches among the representable values, 32 at a time.
  __device__ float edge_of(int b) const {
    const int lane = threadIdx.x & 31;
    uint32_t low = key_of(-INFINITY), high = key_of(weigh.top);  // low's bin is late enough, high's is not
    while (high - low > 1) {
      const uint32_t part = (high - low) / 33 + 1, probe = low + part * (lane + 1);
      const unsigned late = __ballot_sync(0xffffffffu, probe < high && weigh.bin_of(value_of(probe)) >= b);
      const uint32_t n = __popc(late);  // bins fall with the logit: the first n probes
      high = min(high, low + part * (n + 1));
      low += part * n;
    }
    return value_of(low);
  }
  // Lead, all threads: bins sh.lo .. sh.hi as a range of logits.
  __device__ void find_edges() {
    __syncthreads();
    if (threadIdx.x < 32) {
      const float from = sh.lo > 0 ? edge_of(sh.lo) : INFINITY;
      if (threadIdx.x == 0) sh.answer.from = from;
    } else if (threadIdx.x < 64) {
      const float to = edge_of(sh.hi + 1);
      if (threadIdx.x == 32) sh.answer.to = to;
    }
  }

  // A first guess for top-k: of one value per thread, its largest, the want-th is no larger than the
  // row's want-th, and not much smaller as long as the threads outnumber `want`. All tokens above
  // its bin's end are collected then, without a histogram of the row.
  __device__ void guess_from(float largest, u64 want) {
    const int b = weigh.bin_of(largest);
    if (b < BINS - 1) atomicAdd(&reinterpret_cast<uint32_t*>(sh.digits)[b], 1u);
    decide_bins<false>(want, 0.0, true);
  }

  // Which bins the border lies in. `share` of the weight, or `want` tokens.
  template <bool BY_MASS>
  __device__ void find_bins(u64 want, double share, u64 floor) {
    const uint32_t bins = static_cast<uint32_t>(__cvta_generic_to_shared(sh.digits));  // empty since the last barrier
    const float unit = vocab <= WIDE ? 8192.f : 2048.f;                                  // a row's sum stays within 32 bits
    each([&](float x, int i) {
      const float place = weigh.place_of(x), z = __fadd_rd(place, 8388608.f);
      const uint32_t b = __float_as_uint(z) & (BINS - 1);
      bool counts = b != BINS - 1;
      if (floor) counts = counts && order_of(x, i) >= floor;
      // the weight over that at the bin's upper end, a straight line to 2^-15
      const uint32_t w = BY_MASS ? __float_as_uint(fmaf(place - (z - 8388608.f), -0.00742f * unit, unit + 8388608.f)) & 0x3fffu : 1u;
      // predicated, no branch: the values' arithmetic stays one block
      asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p red.shared.add.u32 [%0], %1;\n\t}" ::"r"(bins + b * 4), "r"(w), "r"(static_cast<uint32_t>(counts)) : "memory");
    });
    decide_bins<BY_MASS>(want, share, false);
  }
  template <bool BY_MASS>
  __device__ void decide_bins(u64 want, double share, bool guess) {
    const uint32_t* const bins = sum_up(reinterpret_cast<uint32_t*>(sh.digits), BINS);
    if (is_lead()) {
      constexpr int RUN = BINS / THREADS;
      const int b0 = threadIdx.x * RUN;
      uint32_t here[RUN];
#pragma unroll
      for (int i = 0; i < RUN; ++i) here[i] = bins[b0 + i];
      if (threadIdx.x == 0) {
        sh.answer.verdict = BY_MASS ? FOUND : NOTHING;
        sh.lo = 0;
        sh.hi = BINS - 2;
      }
      if (BY_MASS) {
        float mine = 0.f, all;
        const float first = exp2f(-static_cast<float>(b0) / BINS_PER_OCTAVE);
        auto weight_in = [&](int i) { return static_cast<float>(here[i]) * (first * (1.f - i * 0.00742f + i * i * 2.75e-5f)); };  // 2^(-i / 93)
#pragma unroll
        for (int i = 0; i < RUN; ++i) mine += weight_in(i);
        float sum = block_before(mine, reinterpret_cast<float*>(sh.red), all);
        // each token is rounded to half a unit, either way, on a line that is good to 2^-15: so are sums
        const float slack = vocab <= WIDE ? 0x1.8p-14f : 0x1.2p-12f;
        const float low = static_cast<float>(share) * all * (1 - slack), high = static_cast<float>(share) * all * (1 + slack);
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
          const float next = sum + weight_in(i);
          if (sum < low && low <= next) sh.lo = b0 + i;
          if (sum < high && high <= next) sh.hi = b0 + i;
          sum = next;
        }
      } else {
        u64 mine = 0, all;
#pragma unroll
        for (int i = 0; i < RUN; ++i) mine += here[i];
        u64 sum = block_before(mine, sh.red, all);
        if (sum < want && want <= sum + mine) {
#pragma unroll
          for (int i = 0; i < RUN; ++i) {
            if (sum < want && want <= sum + here[i]) {
              // when all that may stay fits the list, it is collected from the first bin on
              const bool fits = guess || sum + here[i] <= LIST;
              sh.lo = fits ? 0 : b0 + i;
              sh.hi = b0 + i;
              sh.answer.want = want - sum;
              sh.answer.verdict = fits ? ALL_LISTED : FOUND;
            }
            sum += here[i];
          }
        }
      }
      find_edges();
    }
    tell();
  }

  // A candidate goes to the CTA's list; more than LIST are only counted.
  __device__ __forceinline__ void collect(u64 order) {
    const int at = atomicAdd(&sh.listed, 1);
    if (at < LIST) sh.list[at] = order;
  }
  // After everybody collected: the candidates' number, and the lead has them if they fit its list.
  // Contains a barrier, and another must follow before a list is used again.
  __device__ __forceinline__ int gather() {
    __syncthreads();
    if (threadIdx.x < ctas) cluster.map_shared_rank(&sh, threadIdx.x)->counts[rank] = sh.listed;
    cluster.sync();
    int n = 0;
    for (int c = 0; c < ctas; ++c) n = min(n + sh.counts[c], 2 * LIST);
    if (is_lead() && n <= LIST)
      for (int i = sh.counts[0] + threadIdx.x; i < n; i += THREADS) {
        int c = 0, at = i;
        while (at >= sh.counts[c]) at -= sh.counts[c++];
        sh.list[i] = cluster.map_shared_rank(&sh, c)->list[at];
      }
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    return n;
  }

  // Lead: the list in falling order (many: bitonic; a thread has a pair, and pairs less than 64 places apart
  // are a warp's own).
  __device__ void sort_list(int n) {
    if (n <= 128) {  // few: each counts those before it
      u64 o = 0;
      int place = 0;
      if (threadIdx.x < n) {
        o = sh.list[threadIdx.x];
#pragma unroll 8
        for (int i = 0; i < n; ++i) place += sh.list[i] > o || (sh.list[i] == o && i < threadIdx.x);
      }
      __syncthreads();
      if (threadIdx.x < n) sh.list[place] = o;
      __syncthreads();
      return;
    }
    int size = 2;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += THREADS) sh.list[i] = 0;
    __syncthreads();
    const int t = threadIdx.x;
    for (int block = 2; block <= size; block *= 2)
      for (int stride = block / 2; stride > 0; stride /= 2) {
        if (t < size / 2) {
          const int i = 2 * t - (t & (stride - 1)), j = i + stride;
          const u64 a = sh.list[i], b = sh.list[j];
          if ((a < b) == ((i & block) == 0)) {
            sh.list[i] = b;
            sh.list[j] = a;
          }
        }
        if (stride > 32 || (stride == 1 && block >= 64)) __syncthreads();
        else __syncwarp();
      }
    __syncthreads();
  }
  __device__ __forceinline__ u64 weight_of(u64 order) const { return weigh.whole(value_of(static_cast<uint32_t>(order >> INDEX_BITS))); }

  // Lead: sorts the list and finds the place at which the running count or weight reaches `want`;
  // returns the list's whole count or weight, which `want` may be beyond.
  template <bool BY_MASS>
  __device__ u64 rank_list(int n, u64 want) {
    u64 all = n;
    sort_list(n);
    if (!BY_MASS) {
      if (threadIdx.x == 0) sh.answer.border = sh.list[want - 1];
    } else {
      const int c = 2 * threadIdx.x;
      const u64 w0 = c < n ? weight_of(sh.list[c]) : 0, w1 = c + 1 < n ? weight_of(sh.list[c + 1]) : 0;
      const u64 before = block_before(w0 + w1, sh.red, all);
      if (before < want && want <= before + w0) sh.answer.border = sh.list[c];
      else if (before + w0 < want && want <= before + w0 + w1) sh.answer.border = sh.list[c + 1];
    }
    __syncthreads();
    return all;
  }

  // Lead: the list holds everything that top-k may keep. The rest of the row's work is done on it.
  __device__ void draw_from_list(int n, int64_t k, float top_p, u64 least, float u, const SampleParams& p, int r) {
    const int c = 2 * threadIdx.x;
    sort_list(n);
    u64 order[2], w[2], all;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      order[q] = c + q < n ? sh.list[c + q] : 0;
      w[q] = c + q < n && c + q < k ? weight_of(order[q]) : 0;
    }
    u64 ahead = block_before(w[0] + w[1], sh.red, all);
    const u64 need = top_p < 1.f ? share_of(top_p, all) : ~0ull;
    u64 total = 0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const u64 mine = w[q];
      if (ahead >= need || mine < least) w[q] = 0;
      ahead += mine;
      if (c + q < LIST) sh.mass[c + q] = w[q];
      total += w[q];
      // what stays, again, by rising index; 20 bits of it above the place its weight is kept at
      if (c + q < n) sh.list[c + q] = w[q] ? 1ull << 40 | (order[q] & (MAX_VOCAB - 1)) << 12 | (c + q) : 0;
    }
    total = block_total(total, sh.red);
    sort_list(n);
    const u64 target = target_of(u, total);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      order[q] = c + q < n ? sh.list[c + q] : 0;
      w[q] = order[q] ? sh.mass[order[q] & 0xfff] : 0;
    }
    u64 before = block_before(w[0] + w[1], sh.red, all);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (before <= target && target < before + w[q]) finish(p, r, index_of(order[q] >> 12), log_share(w[q], total));
      before += w[q];
    }
  }

  // More candidates than the list takes: narrow them by digits of the order, largest first.
  // Candidates are tokens with logits in (to, from], at or above `floor`; answer.want says how far in
  // the border is.
  template <bool BY_MASS>
  __device__ u64 narrow(u64 floor) {
    const float from = sh.answer.from, to = sh.answer.to;
    u64 prefix = 0, mask = 0;
    for (int shift = INDEX_BITS + 32 - DIGIT_BITS;;) {
      auto candidate = [&](float x, int i, u64& o) {
        o = order_of(x, i);
        return x > to && x <= from && o >= floor && (o & mask) == prefix;
      };
      each([&](float x, int i) {
        u64 o;
        if (candidate(x, i, o)) atomicAdd(&sh.digits[DIGITS - 1 - (static_cast<int>(o >> shift) & (DIGITS - 1))], BY_MASS ? weigh.whole(x) : 1);
      });
      const u64* const sums = sum_up(sh.digits, DIGITS);
      if (is_lead()) {
        constexpr int RUN = DIGITS / THREADS;
        const int d0 = threadIdx.x * RUN;
        const u64 want = sh.answer.want;
        u64 mine = 0, all;
#pragma unroll
        for (int i = 0; i < RUN; ++i) mine += sums[d0 + i];
        u64 sum = block_before(mine, sh.red, all);
        if (sum < want && want <= sum + mine) {  // one thread: want is at most the candidates' sum
          int d = d0;
          while (want > sum + sums[d]) sum += sums[d++];
          sh.answer.prefix = prefix | static_cast<u64>(DIGITS - 1 - d) << shift;
          sh.answer.want = want - sum;
        }
      }
      tell();
      prefix = sh.answer.prefix;
      mask |= static_cast<u64>(DIGITS - 1) << shift;
      each([&](float x, int i) {
        u64 o;
        if (candidate(x, i, o)) collect(o);
      });
      const int n = gather();
      if (is_lead() && n <= LIST) rank_list<BY_MASS>(n, sh.answer.want);
      tell();
      if (n <= LIST) return sh.answer.border;
      shift = shift > DIGIT_BITS ? shift - DIGIT_BITS : 0;  // at 0 the whole place is known: one candidate
    }
  }

  // Lead: which run lies `target` into the runs' weights (or counts).
  __device__ void locate(u64 before, u64 w, u64 target, u64 total) {
    if (before <= target && target < before + w) {
      sh.answer.owner = threadIdx.x;
      sh.answer.residual = target - before;
      sh.answer.total = total;
    }
  }
  __device__ void locate(float u) {
    const u64 w = threadIdx.x < ctas * WARPS ? sh.kept[threadIdx.x] : 0;
    u64 total;
    const u64 before = block_before(w, sh.red, total);
    locate(before, w, target_of(u, total), total);
  }

  // The CTA that has the owner's run goes through it together.
  template <typename W>
  __device__ void draw(const SampleParams& p, int r, W weight) {
    const int owner = sh.answer.owner;
    if (owner / WARPS != rank) return;
    const int from = owner == 0 ? 0 : min(tail, head + owner * run_length()), to = owner == runs() - 1 ? vocab : min(tail, head + (owner + 1) * run_length());
    const u64 residual = sh.answer.residual;
    u64 sum = 0;
    for (int j = from; j < to && sum <= residual; j += THREADS) {
      const int i = j + threadIdx.x;
      const u64 w = i < to ? weight(as_f32(row[i]), i) : 0;
      u64 all;
      const u64 before = sum + block_before(w, sh.red, all);
      if (before <= residual && residual < before + w) finish(p, r, i, log_share(w, sh.answer.total));
      sum += all;
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(THREADS, CTAS_PER_SM) sample_kernel(const SampleParams p) {
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();  // waited for below: nobody writes to a CTA that has not started
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int r = blockIdx.x / ctas;
  const int run = rank * WARPS + warp;  // index order is: run, then within it
  Sampler<T> me{cluster, sh, *cluster.map_shared_rank(&sh, 0), static_cast<const T*>(p.logits) + r * p.row_stride, run, ctas, rank, p.vocab, p.steps};
  me.cut();

  // ---- the maximum (fmaxf passes NaN over)
  float top = -INFINITY;
  me.each([&](float x, int) { top = fmaxf(top, x); });
  {
    constexpr int MINE = TABLE * COPIES / THREADS;  // copies of one value, by each thread
    const double value = exp2(static_cast<double>(tid * MINE / COPIES) / TABLE) * WEIGHT_ONE;
#pragma unroll
    for (int i = 0; i < MINE; ++i) sh.table[tid * MINE + i] = value;
  }
  me.clear_bins();
  if (tid == 0) sh.listed = 0;
  const float temperature = p.temperature ? p.temperature[r * p.st] : 1.f;
  const float top_p = p.top_p ? p.top_p[r * p.sp] : 1.f;
  const float min_p = p.min_p ? p.min_p[r * p.sm] : 0.f;
  const float u = p.uniform[r * p.su];
  const int64_t k = p.top_k ? (p.k64 ? static_cast<const int64_t*>(p.top_k)[r * p.sk] : static_cast<const int32_t*>(p.top_k)[r * p.sk]) : 0;
  const float mine_top = top;
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  float* const redf = reinterpret_cast<float*>(sh.red);
  if (lane == 0) redf[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) top = fmaxf(top, redf[w]);
  cluster.barrier_wait();
  if (tid < ctas) cluster.map_shared_rank(&sh, tid)->tops[rank] = top;
  cluster.sync();
  for (int c = 0; c < ctas; ++c) top = fmaxf(top, sh.tops[c]);

  if (top == -INFINITY) {
    if (rank == 0 && tid == 0) finish(p, r, -1, -INFINITY);
    return;
  }
  if (!(temperature > 0.f) || k == 1 || top_p <= 0.f) {  // the first of the largest
    int at = p.vocab;
    me.each([&](float x, int i) {
      if (x == top) at = min(at, i);
    });
#pragma unroll
    for (int d = 16; d; d >>= 1) at = min(at, __shfl_xor_sync(0xffffffffu, at, d));
    int* const redi = reinterpret_cast<int*>(sh.red);
    __syncthreads();
    if (lane == 0) redi[warp] = at;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) at = min(at, redi[w]);
    if (tid == 0) me.lead.firsts[rank] = at;
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int c = 0; c < ctas; ++c) at = min(at, sh.firsts[c]);
      finish(p, r, at, 0.f);
    }
    return;
  }
  if (top == INFINITY) {  // tokens at +inf share the weight, nothing else has any
    int n = 0;
    me.each([&](float x, int) { n += x == INFINITY; });
    n = warp_total(n);
    if (lane == 0) me.lead.kept[run] = n;
    cluster.sync();
    if (me.is_lead()) {
      const u64 w = tid < ctas * WARPS ? sh.kept[tid] : 0;
      u64 all;
      const u64 before = block_before(w, sh.red, all);
      if (k > 0 && static_cast<u64>(k) < all) all = static_cast<u64>(k);
      if (top_p < 1.f) all = max(share_of(top_p, all), 1ull);
      me.locate(before, w, target_of(u, all), all);
    }
    me.tell();
    me.draw(p, r, [](float x, int) -> u64 { return x == INFINITY; });
    return;
  }

  Weighing& weigh = me.weigh;
  weigh.top = top;
  weigh.half_top = 0.5f * top;
  weigh.bin_scale = fminf(2.f * BINS_PER_OCTAVE * 1.44269504f / temperature, 3e38f);
  weigh.top64 = static_cast<double>(top);
  weigh.scale = TABLE * 1.4426950408889634073599 / static_cast<double>(temperature);
  // 2^-43 of the largest, rounded down: a whole weight of zero there, and above it at least 2^-43. (Below
  // the maximum also where that many units are lost in its last place.)
  weigh.lowest = fminf(__double2float_rd(weigh.top64 - (WEIGHT_BITS + 1) * 0.69314718055994530942 * static_cast<double>(temperature)), nextafterf(top, -INFINITY));
  weigh.table = sh.table + lane % COPIES;
  const u64 least = min_p > 0.f ? __double2ull_ru(fmin(static_cast<double>(min_p), 1.0) * static_cast<double>(WEIGHT_ONE)) : 0;
  u64 border = 0;
  bool have_runs = false;  // the answer already says which run the draw lies in

  if (k > 0 && k < p.vocab) {
    bool guess = k <= LIST / 2 && k <= ctas * THREADS / 4;
    if (guess) me.guess_from(mine_top, static_cast<u64>(k));
    for (;; guess = false) {
      if (!guess) me.template find_bins<false>(static_cast<u64>(k), 0.0, 0);
      if (sh.answer.verdict == NOTHING) {  // among weights of zero; or too few threads have anything, which says nothing of the row
        if (guess) continue;
        break;
      }
      const float from = sh.answer.from, to = sh.answer.to;
      const bool all = sh.answer.verdict == ALL_LISTED;
      me.each([&](float x, int i) {
        if (x > to && x <= from) me.collect(order_of(x, i));
      });
      const int n = me.gather();
      if (all && n <= LIST) {
        // nothing is asked of the other CTAs any more, once the lead has read their lists
        cluster.barrier_arrive();
        if (me.is_lead()) me.draw_from_list(n, k, top_p, least, u, p, r);
        cluster.barrier_wait();
        return;
      }
      if (all) {  // the guess was too low
        cluster.sync();
        continue;
      }
      if (me.is_lead() && n <= LIST) me.template rank_list<false>(n, sh.answer.want);
      me.tell();
      border = n <= LIST ? sh.answer.border : me.template narrow<false>(0);
      break;
    }
  }
  if (top_p < 1.f) {
    me.template find_bins<true>(0, static_cast<double>(top_p), border);
    do {
      const float from = sh.answer.from, to = sh.answer.to;
      Tally all, before;
      me.each([&](float x, int i) {
        if (border && order_of(x, i) < border) return;
        const double w = weigh.of(x);
        if (weigh.counts(x)) all.add(w);
        if (x > from) before.add(w);
        else if (x > to) me.collect(order_of(x, i));
      });
      const u64 a = warp_total(before.value()), z = warp_total(all.value());
      if (lane == 0) {
        me.lead.kept[run] = a;
        me.lead.all[run] = z;
      }
      const int n = me.gather();
      if (n > LIST) {  // their weight, which else the ranked list gives
        u64 m = 0;
        me.each([&](float x, int i) {
          if (x > to && x <= from && !(border && order_of(x, i) < border)) m += weigh.whole(x);
        });
        m = warp_total(m);
        if (lane == 0) me.lead.middle[run] = m;
        cluster.sync();
      }
      if (me.is_lead()) {
        // the sums are few enough for every warp to add them up itself
        u64 a = 0, z = 0, m = 0;
        for (int c = lane; c < me.runs(); c += 32) {
          a += sh.kept[c];
          z += sh.all[c];
          if (n > LIST) m += sh.middle[c];
        }
        a = warp_total(a);
        z = warp_total(z);
        m = warp_total(m);
        const u64 need = share_of(top_p, z);
        if (a < need && n <= LIST) m = me.template rank_list<true>(n, need - a);
        const bool right = a < need && need <= a + m;
        if (right && n <= LIST) {
          const u64 found = sh.answer.border;
          for (int c = tid; c < n; c += THREADS)
            if (sh.list[c] >= found) atomicAdd(&sh.kept[me.run_of(index_of(sh.list[c]))], me.weight_of(sh.list[c]));
          __syncthreads();
          me.locate(u);
        }
        __syncthreads();
        if (tid == 0) {
          sh.answer.verdict = !right ? WRONG_BINS : n <= LIST ? FOUND : TOO_MANY;
          sh.answer.want = need - a;
          sh.lo = 0;  // should the exact sums say that the border is elsewhere: every bin
          sh.hi = BINS - 2;
        }
        if (!right) me.find_edges();
      }
      me.tell();
    } while (sh.answer.verdict == WRONG_BINS);
    have_runs = sh.answer.verdict == FOUND && !least;
    border = sh.answer.verdict == FOUND ? sh.answer.border : me.template narrow<true>(border);
  }
  auto kept_weight = [&](float x, int i) -> u64 {
    if (border && order_of(x, i) < border) return 0;
    const u64 w = weigh.whole(x);
    return w >= least ? w : 0;  // the largest weighs 2^42: it always stays
  };
  if (!have_runs) {
    u64 mine = 0;
    if (border || least) {
      me.each([&](float x, int i) { mine += kept_weight(x, i); });
    } else {
      Tally all;
      me.each([&](float x, int) {
        const double w = weigh.of(x);
        if (weigh.counts(x)) all.add(w);
      });
      mine = all.value();
    }
    mine = warp_total(mine);
    if (lane == 0) me.lead.kept[run] = mine;
    cluster.sync();
    if (me.is_lead()) me.locate(u);
    me.tell();
  }
  me.draw(p, r, kept_weight);
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
  for (const lh_memref_t* m : {tokens, logprobs, logits, uniform, temperature, top_k, top_p, min_p})
    if (m && reinterpret_cast<uintptr_t>(data_ptr(m)) % dtype_size(m->dtype)) return set_error(ctx, LH_ERR_INVALID, "sample: an operand is not aligned to its type");
  for (const lh_memref_t* m : {tokens, logprobs})
    if (m && n > 1 && m->strides[0] == 0) return set_error(ctx, LH_ERR_INVALID, "sample: a written operand overlaps itself (zero stride)");
  if (n == 0) return LH_OK;
  SampleParams p;
  memset(&p, 0, sizeof(p));
  p.logits = data_ptr(logits); p.row_stride = logits->strides[0];
  p.vocab = static_cast<int>(v);
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
  // How many CTAs share a row, measured with top-p over 131071 f32 logits. One row ends soonest on eight, the
  // largest cluster that every launch may have (89 us on one CTA, 57 on two, 40 on four, 32 on eight), but more
  // CTAs than are resident at once wait for one another's clusters: 64 rows take 69 us on two, 57 on four, 71 on
  // eight; 256 rows 170 on one, 172 on two, 196 on four. Rows of a few values per thread take fewer.
  const int64_t vec = 16 / static_cast<int64_t>(dtype_size(logits->dtype));
  const int64_t groups = v / vec > 0 ? v / vec : 1;  // whole ones; the odd ends are the first and the last warp's
  const int64_t resident = static_cast<int64_t>(ctx->sm_count) * CTAS_PER_SM;
  int ctas = groups > THREADS ? 2 : 1;
  while (ctas > 1 && ctas < MAX_CLUSTER && groups > static_cast<int64_t>(ctas) * THREADS && n * ctas * 2 <= resident) ctas *= 2;
  p.steps = static_cast<int>((groups + static_cast<int64_t>(ctas) * THREADS - 1) / (static_cast<int64_t>(ctas) * THREADS));
  if (n > 0x7fffffffll / ctas) return set_error(ctx, LH_ERR_UNSUPPORTED, "sample: %lld rows are too many for one call", (long long)n);
  DeviceScope scope(ctx->device);
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(n * ctas));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LH_CUDA_CHECK(ctx, cudaLaunchKernelEx(&cfg, logits->dtype == LH_F32 ? sample_kernel<float> : logits->dtype == LH_BF16 ? sample_kernel<__nv_bfloat16> : sample_kernel<__half>, p));
  LH_CHECK_LAUNCH(ctx, "sample_kernel");
  return LH_OK;
}
