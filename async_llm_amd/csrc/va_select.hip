// What stays of blocks of tokens: the first and the last few of a block, and of the others the heaviest.
//
//   score(t) = fp32(sum over kv heads, in 64 bits, of weights[h][slots[t]])
//   kept     = the `keep` largest by (protected, score, -t), in rising order of t
//
// Scores become 32-bit keys whose order as whole numbers is theirs (protected tokens above all, NaN next); the keep-th largest key
// is found digit by digit from histograms, most significant first, and then every token above it stays, and of those equal to
// it the first that are wanted.  No sort, and no order of execution that the result depends on.
//
// Blocks of up to kSelectInLds tokens: a workgroup each, keys in LDS, one launch (of 4 heads: 8192 tokens 16.7 us, 20.3 by runs, 12000
// 21.7 and 20.7; 64 blocks of 8192 18.4 and 23.5, of 12000 24.1 and 25.3; of 16 heads 21.4 and 22.6, 28.9 and 23.1).  Longer ones: four
// launches of a workgroup for each run of tokens.  The first makes keys and counts those of a run by their upper digit; each
// further one adds the counts of all runs up, every workgroup for itself, finds the cut's digit, and counts the run's keys that have it
// by their next one, and the last writes.  What lies above the cut in the runs in front falls out of the same sums.  They are
// taken of groups of 32 digits first, then of the one group that has the cut: 29 us instead of 41 with all of them, for an eighth of 8
// blocks of 60000 to 131072 tokens.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "va_device.h"
#include "va_internal.h"
#include "va_launch.h"

namespace va {

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / kWave;
constexpr int kSelectInLds = 10240;  // tokens of a block whose keys stay in LDS
constexpr int kSelectBlocks = 64;    // blocks of a launch
constexpr int kSelectRun = 4096;     // tokens of a run, at least
constexpr int kSelectBins = 256;
// digits of a long block's keys: eleven bits, eleven, ten; counts of a run by each, and of groups of 32 neighbouring ones
constexpr int kSelectTop = 2048, kSelectGroup = 32, kSelectGroupsAt = 5120, kSelectCounts = kSelectGroupsAt + 5120 / kSelectGroup;

struct SelectBlock {
  long long begin, out;  // first entry of its slots, of its results
  long long count, keep;
  long long keys;  // long blocks: first key in the workspace
  int runs, first_run, run_tokens;  // long blocks: runs, number of the first one in the workspace, tokens of a run
};
struct SelectArgs {
  const float* weights;
  long long num_slots;
  int num_heads;
  const int64_t* slots;
  long long first, last;  // tokens protected at both ends
  int64_t* positions;
  int64_t* out_slots;
  int64_t* shifts;
  // long blocks
  uint32_t* keys;
  uint32_t* found;   // [block][2 stages][2]: the cut's digits so far, how many of the keys with them are wanted
  uint32_t* before;  // [run][2 stages]: tokens of the runs in front of it that are above the cut in this stage's digit
  uint32_t* counts;  // [run][kSelectCounts]: tokens by the upper digit of their keys, of those with the cut's by the middle one, then by the lower one;
                     // then the same by groups of digits
  SelectBlock blocks[kSelectBlocks];
};

__device__ __forceinline__ uint32_t key_of(float score) {
  if (score != score) return 0xfffffffeu;
  const uint32_t bits = __float_as_uint(score + 0.f);  // (-0 counts as 0)
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// Keys of tokens [begin, end) of a block, this thread's every kSelectThreads-th: `put(t, key)`.  A slot and its weights are two trips to
// memory; those of kBatch tokens are made together.
template <typename Put>
__device__ __forceinline__ void make_keys(const SelectArgs& a, const SelectBlock& b, long long begin, long long end, Put&& put) {
  constexpr int kBatch = 4, kHeads = 4;
  for (long long t0 = begin + threadIdx.x; t0 < end; t0 += kBatch * kSelectThreads) {
    long long slot[kBatch];
    bool protect[kBatch];
    double sum[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const long long t = min(t0 + u * kSelectThreads, end - 1);
      protect[u] = t < a.first || t >= b.count - a.last;
      slot[u] = a.slots[b.begin + t];
      sum[u] = 0.0;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (slot[u] < 0 || slot[u] >= a.num_slots) slot[u] = -1;
    for (int h0 = 0; h0 < a.num_heads; h0 += kHeads) {
      float w[kBatch][kHeads];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
#pragma unroll
        for (int i = 0; i < kHeads; ++i) w[u][i] = a.weights[min(h0 + i, a.num_heads - 1) * a.num_slots + max(slot[u], 0ll)];
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if (h0 + i < a.num_heads && slot[u] >= 0) sum[u] += (double)w[u][i];
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const long long t = t0 + u * kSelectThreads;
      if (t < end) put(t, protect[u] ? 0xffffffffu : key_of((float)sum[u]));
    }
  }
}

// Scores of tokens that nobody looked at are equal, and most others share a few upper digits: lanes count in sixteen copies, or adds
// to one bin would take a clock each.
constexpr int kSelectCopies = 16;

// The keep-th largest of `count` keys, or a number below it that is above all that do not stay, and how many of the keys equal to
// it are among the first `keep`; 1 <= keep <= count.  All threads of the workgroup call it and get the same.
struct Cut {
  uint32_t key, equal;
};
template <typename Keys>
__device__ __forceinline__ Cut find_cut(Keys key_at, long long count, long long keep, uint32_t (&bins)[kSelectBins * kSelectCopies],
                                        uint32_t (&found)[3]) {
  uint32_t prefix = 0, wanted = (uint32_t)keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < kSelectBins * kSelectCopies; i += kSelectThreads) bins[i] = 0;
    __syncthreads();
    for (long long t = threadIdx.x; t < count; t += kSelectThreads) {
      const uint32_t key = key_at(t);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&bins[((key >> shift) & 255u) * kSelectCopies + threadIdx.x % kSelectCopies], 1u);
    }
    __syncthreads();
    // thread 4 d + i: four copies of digit d
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) mine += bins[threadIdx.x * 4 + i];
    mine += __shfl_xor(mine, 1, kWave);
    mine += __shfl_xor(mine, 2, kWave);
    __syncthreads();
    if (threadIdx.x % 4 == 0) bins[threadIdx.x / 4] = mine;
    __syncthreads();
    if (threadIdx.x < kWave) {  // lane l: digits 4 l .. + 3; the digit is where the count from above reaches `wanted`
      const int lane = threadIdx.x;
      uint32_t n[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += n[i] = bins[4 * lane + i];
      uint32_t above = sum;  // of this lane's digits and all higher ones
#pragma unroll
      for (int off = 1; off < kWave; off <<= 1) {
        const uint32_t other = __shfl_down(above, off, kWave);
        if (lane + off < kWave) above += other;
      }
      uint32_t higher = above - sum;
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        if (higher < wanted && higher + n[i] >= wanted) found[0] = 4 * lane + i, found[1] = wanted - higher, found[2] = n[i];
        higher += n[i];
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    wanted = found[1];
    if (found[2] == wanted) return Cut{prefix, ~0u};  // all keys with these digits stay (1500 tokens of 8 heads: 9.4 -> 8.4 us)
  }
  return Cut{prefix, wanted};
}

__device__ __forceinline__ uint32_t bits_below(unsigned long long mask, int lane) { return (uint32_t)__popcll(mask & ((1ull << lane) - 1)); }

// Write those of tokens [begin, end) of a block that stay; a wave's part, four times 64 tokens at a time, whose slots are on their way
// together.  `taken`: kept tokens in front of it, `equal`: tokens equal to the cut's key in front of it.
template <typename Keys>
__device__ __forceinline__ void write_kept(const SelectArgs& a, const SelectBlock& b, Keys key_at, Cut cut, long long begin, long long end,
                                           uint32_t taken, uint32_t equal) {
  constexpr int kBatch = 4;
  const int lane = threadIdx.x % kWave;
  for (long long t0 = begin; t0 < end; t0 += kBatch * kWave) {
    uint32_t key[kBatch];
    int64_t slot[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const long long t = min(t0 + u * kWave + lane, end - 1);
      key[u] = key_at(t);
      slot[u] = a.slots[b.begin + t];
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const long long t = t0 + u * kWave + lane;
      const bool same = t < end && key[u] == cut.key;
      const unsigned long long sames = __ballot(same);
      const bool stays = t < end && (key[u] > cut.key || (same && equal + bits_below(sames, lane) < cut.equal));
      const unsigned long long kept = __ballot(stays);
      if (stays) {
        const long long rank = (long long)taken + bits_below(kept, lane), at = b.out + rank;
        a.positions[at] = t;
        a.out_slots[at] = slot[u];
        a.shifts[at] = rank - t;
      }
      equal += (uint32_t)__popcll(sames);
      taken += (uint32_t)__popcll(kept);
    }
  }
}

__global__ __launch_bounds__(kSelectThreads) void select_kernel(SelectArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t bins[kSelectBins * kSelectCopies], found[3], of_wave[kSelectWaves][2];
  const SelectBlock& b = a.blocks[blockIdx.x];
  if (b.keep == 0) return;
  const int count = (int)b.count;
  make_keys(a, b, 0, count, [&](long long t, uint32_t key) __attribute__((always_inline)) { keys[t] = key; });
  __syncthreads();
  auto key_at = [&](long long t) __attribute__((always_inline)) { return keys[t]; };
  const Cut cut = find_cut(key_at, count, b.keep, bins, found);
  // each wave a run of tokens: how many stay before it, then it writes
  const int wave = threadIdx.x / kWave, each = (count + kSelectThreads - 1) / kSelectThreads * kWave;
  const int begin = min(wave * each, count), end = min(begin + each, count);
  uint32_t above = 0, same = 0;
  for (int t0 = begin; t0 < end; t0 += kWave) {
    const int t = t0 + threadIdx.x % kWave;
    const uint32_t key = t < end ? keys[t] : 0u;
    above += (uint32_t)__popcll(__ballot(t < end && key > cut.key));
    same += (uint32_t)__popcll(__ballot(t < end && key == cut.key));
  }
  if (threadIdx.x % kWave == 0) of_wave[wave][0] = above, of_wave[wave][1] = same;
  __syncthreads();
  above = same = 0;
  for (int w = 0; w < wave; ++w) above += of_wave[w][0], same += of_wave[w][1];
  write_kept(a, b, key_at, cut, begin, end, above + min(same, cut.equal), same);
}

// ---- long blocks ----
// Sums over the runs of kDigits neighbouring counts from `from`, those of a run kSelectCounts apart, from above: the digit at which they
// reach `wanted`, what is then still wanted, and the counts in front of this run above that digit and at it.  All threads call it and get the same.
struct Digit {
  uint32_t digit, wanted, above, at;
};
template <int kDigits>
__device__ __forceinline__ Digit find_digit(const uint32_t* from, int runs, int run, uint32_t wanted, uint32_t (&sums)[2][kSelectWaves][kWave], uint32_t (&found)[4]) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, digit = kDigits - 1 - threadIdx.x % kDigits;
  uint32_t n = 0, front = 0;
#pragma unroll 4
  for (int r = threadIdx.x / kDigits; r < runs; r += kSelectThreads / kDigits) {
    const uint32_t x = from[(long long)r * kSelectCounts + digit];
    n += x, front += r < run ? x : 0u;
  }
  if constexpr (kDigits == 32) n += __shfl_xor(n, 32, kWave), front += __shfl_xor(front, 32, kWave);
  sums[0][wave][lane] = n, sums[1][wave][lane] = front;
  __syncthreads();
  if (wave == 0) {
    n = front = 0;
#pragma unroll
    for (int w = 0; w < kSelectWaves; ++w) n += sums[0][w][lane], front += sums[1][w][lane];
    if (lane >= kDigits) n = front = 0;
    uint32_t upto = n, fronts = front;  // with all that is above
#pragma unroll
    for (int off = 1; off < kDigits; off <<= 1) {
      const uint32_t other = __shfl_up(upto, off, kWave), others = __shfl_up(fronts, off, kWave);
      if (lane >= off) upto += other, fronts += others;
    }
    if (lane < kDigits && upto - n < wanted && upto >= wanted) found[0] = (uint32_t)digit, found[1] = wanted - (upto - n), found[2] = fronts - front, found[3] = front;
  }
  __syncthreads();
  const Digit d{found[0], found[1], found[2], found[3]};
  __syncthreads();
  return d;
}

// Stage 0: keys, counted by their upper digit.  Stage 1 (2): the cut's upper (middle) digit, the run's keys that have it counted by
// the next one.  Stage 3: the lower digit, and the run writes what stays.
template <int kStage>
__global__ __launch_bounds__(kSelectThreads) void select_run_kernel(SelectArgs a) {
  constexpr int kDigits = kStage == 3 ? 1024 : kSelectTop;  // of the digit that is found
  constexpr int kNext = kStage == 2 ? 1024 : kSelectTop, kCopies = 4;  // of the one that is counted
  constexpr int kFrom = kStage == 1 ? 0 : kStage == 2 ? 2048 : 4096, kTo = kStage == 0 ? 0 : kStage == 1 ? 2048 : 4096;
  __shared__ uint32_t bins[kStage == 3 ? 1 : kCopies][kStage == 3 ? 1 : kNext + 8];
  __shared__ uint32_t sums[2][kSelectWaves][kWave], found[4], per_wave[kSelectWaves][2];
  const SelectBlock& b = a.blocks[blockIdx.y];
  const int run = (int)blockIdx.x;
  if (run >= b.runs) return;
  const long long begin = (long long)run * b.run_tokens, end = min(begin + b.run_tokens, b.count);
  uint32_t* keys = a.keys + b.keys;
  if constexpr (kStage < 3) {
    for (int i = threadIdx.x; i < kCopies * (kNext + 8); i += kSelectThreads) bins[0][i] = 0;
    __syncthreads();
  }
  // this thread's keys: every kStep-th from `from`; the first ones are asked for at once
  constexpr int kAhead = 4, kStep = kStage == 3 ? kWave : kSelectThreads;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const long long each = b.run_tokens / kSelectWaves;
  const long long from = kStage == 3 ? min(begin + wave * each, end) : begin, to = kStage == 3 ? min(from + each, end) : end;
  const long long t0 = from + threadIdx.x % kStep;
  uint32_t first[kAhead];
  if constexpr (kStage > 0)
#pragma unroll
    for (int u = 0; u < kAhead; ++u) first[u] = t0 + u * kStep < to ? keys[t0 + u * kStep] : 0u;
  auto each_key = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (t0 + u * kStep < to) f(first[u]);
#pragma unroll 4
    for (long long t = t0 + kAhead * kStep; t < to; t += kStep) f(keys[t]);
  };
  uint32_t prefix = 0, equal = 0, above = 0, same = 0;
  if constexpr (kStage > 0) {
    const uint32_t* last = a.found + 4 * blockIdx.y + 2 * (kStage - 2);
    const uint32_t* counts = a.counts + (long long)b.first_run * kSelectCounts;
    const Digit group = find_digit<kDigits / kSelectGroup>(counts + kSelectGroupsAt + kFrom / kSelectGroup, b.runs, run, kStage == 1 ? (uint32_t)b.keep : last[1], sums, found);
    const Digit d = find_digit<kSelectGroup>(counts + kFrom + group.digit * kSelectGroup, b.runs, run, group.wanted, sums, found);
    prefix = (kStage == 1 ? 0u : last[0]) | (group.digit * kSelectGroup + d.digit) << (kStage == 1 ? 21 : kStage == 2 ? 10 : 0);
    equal = d.wanted, above = group.above + d.above, same = d.at;
    if constexpr (kStage < 3) {
      if (threadIdx.x == 0) {
        a.before[2 * (b.first_run + run) + kStage - 1] = above;
        if (run == 0) a.found[4 * blockIdx.y + 2 * (kStage - 1)] = prefix, a.found[4 * blockIdx.y + 2 * (kStage - 1) + 1] = equal;
      }
    } else {
      above += a.before[2 * (b.first_run + run)] + a.before[2 * (b.first_run + run) + 1];
    }
  }
  if constexpr (kStage < 3) {
    auto count = [&](uint32_t digit) __attribute__((always_inline)) { atomicAdd(&bins[threadIdx.x % kCopies][digit], 1u); };
    if constexpr (kStage == 0) {
      make_keys(a, b, begin, end, [&](long long t, uint32_t key) __attribute__((always_inline)) {
        keys[t] = key;
        count(key >> 21);
      });
    } else {
      each_key([&](uint32_t key) __attribute__((always_inline)) {
        constexpr int kShift = kStage == 1 ? 21 : 10;
        if (key >> kShift == prefix >> kShift) count(kStage == 1 ? key >> 10 & 2047u : key & 1023u);
      });
    }
    __syncthreads();
    uint32_t* counts = a.counts + (long long)(b.first_run + run) * kSelectCounts;
    uint32_t *digits = counts + kTo, *groups = counts + kSelectGroupsAt + kTo / kSelectGroup;
    for (int i = threadIdx.x; i < kNext; i += kSelectThreads) {
      uint32_t sum = 0;
#pragma unroll
      for (int c = 0; c < kCopies; ++c) sum += bins[c][i];
      digits[i] = sum;
#pragma unroll
      for (int off = 1; off < kSelectGroup; off <<= 1) sum += __shfl_xor(sum, off, kWave);
      if (i % kSelectGroup == 0) groups[i / kSelectGroup] = sum;
    }
  } else {
    const Cut cut{prefix, equal};
    // this wave's part of the run, and what stays in front of it
    uint32_t own_above = 0, own_same = 0;
    each_key([&](uint32_t key) __attribute__((always_inline)) { own_above += key > cut.key, own_same += key == cut.key; });
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) own_above += __shfl_xor(own_above, off, kWave), own_same += __shfl_xor(own_same, off, kWave);
    __syncthreads();
    if (lane == 0) per_wave[wave][0] = own_above, per_wave[wave][1] = own_same;
    __syncthreads();
    for (int w = 0; w < wave; ++w) above += per_wave[w][0], same += per_wave[w][1];
    write_kept(a, b, [&](long long t) __attribute__((always_inline)) { return keys[t]; }, cut, from, to, above + min(same, cut.equal), same);
  }
}

// Runs of kSelectRun tokens, or of a multiple of those that makes about 64.
static int run_tokens_of(long long count) { return kSelectRun * (int)std::max<long long>(1, count / (64ll * kSelectRun)); }
static long long runs_of(long long count) { return (count + run_tokens_of(count) - 1) / run_tokens_of(count); }

static int launch_select_batch(SelectArgs& a, int n, bool in_lds, hipStream_t stream) {
  if (n == 0) return VA_OK;
  const dim3 block(kSelectThreads);
  long long most = 0, runs = 0;
  for (int i = 0; i < n; ++i) most = std::max(most, a.blocks[i].count), runs = std::max(runs, (long long)a.blocks[i].runs);
  if (in_lds) {
    static std::atomic<unsigned long long> devices{0};
    const hipError_t e = allow_lds(reinterpret_cast<const void*>(&select_kernel), kSelectInLds * 4, devices);
    if (e != hipSuccess) return va_fail(VA_ERR_HIP, "raising the LDS limit: %s", hipGetErrorString(e));
    hipLaunchKernelGGL(select_kernel, dim3((unsigned)n), block, (unsigned)(most * 4), stream, a);
  } else {
    const dim3 grid((unsigned)runs, (unsigned)n);
    hipLaunchKernelGGL(select_run_kernel<0>, grid, block, 0, stream, a);
    hipLaunchKernelGGL(select_run_kernel<1>, grid, block, 0, stream, a);
    hipLaunchKernelGGL(select_run_kernel<2>, grid, block, 0, stream, a);
    hipLaunchKernelGGL(select_run_kernel<3>, grid, block, 0, stream, a);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "selection launch: %s", hipGetErrorString(e));
}

// Words of the workspace: keys, digits found and counts of all long blocks (batches start on 16-byte boundaries); -1 for counts that no selection takes.
static int64_t select_words(int32_t n_blocks, const int64_t* counts) {
  int64_t words = 0;
  for (int32_t i = 0; i < n_blocks; ++i) {
    if (counts[i] < 0 || counts[i] > 0x7fffffffLL) return -1;
    if (counts[i] > kSelectInLds) words += (counts[i] + 3) / 4 * 4 + 8 + (2 + kSelectCounts) * runs_of(counts[i]);
  }
  return words;
}

}  // namespace va

extern "C" int64_t va_select_workspace_bytes(int32_t n_blocks, const int64_t* counts_host) {
  if (n_blocks < 0 || (n_blocks > 0 && !counts_host)) return -1;
  const int64_t words = va::select_words(n_blocks, counts_host);
  return words < 0 ? -1 : 4 * words;
}

extern "C" int va_select_tokens(const float* weights_dev, int32_t num_heads, int64_t num_slots, const int64_t* slots_dev, int32_t n_blocks,
                                const int64_t* counts_host, const int64_t* keep_host, int64_t first, int64_t last, int64_t* positions_dev,
                                int64_t* out_slots_dev, int64_t* shifts_dev, void* workspace_dev, int64_t workspace_bytes, void* stream) {
  if (n_blocks < 0 || num_heads < 0 || num_slots < 0 || first < 0 || last < 0) return va_fail(VA_ERR_ARG, "negative count");
  if (n_blocks == 0) return VA_OK;
  if (!counts_host || !keep_host) return va_fail(VA_ERR_ARG, "null pointer");
  const int64_t words = va::select_words(n_blocks, counts_host);
  if (words < 0) return va_fail(VA_ERR_ARG, "a block holds 0 to 2^31 - 1 tokens");
  int64_t kept = 0;
  for (int32_t i = 0; i < n_blocks; ++i) {
    if (keep_host[i] < 0 || keep_host[i] > counts_host[i])
      return va_fail(VA_ERR_ARG, "block %d: %lld of %lld tokens cannot stay", (int)i, (long long)keep_host[i], (long long)counts_host[i]);
    kept += keep_host[i];
  }
  if (kept == 0) return VA_OK;
  if ((num_heads && num_slots && !weights_dev) || !slots_dev || !positions_dev || !out_slots_dev || !shifts_dev)
    return va_fail(VA_ERR_ARG, "null pointer");
  if (words && (!workspace_dev || (uintptr_t)workspace_dev % 16)) return va_fail(VA_ERR_ARG, "a selection from long blocks needs a 16-byte aligned workspace");
  if (workspace_bytes < 4 * words)
    return va_fail(VA_ERR_CAPACITY, "workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)(4 * words));
  // both kinds in batches of kSelectBlocks
  for (int large = 0; large < 2; ++large) {
    va::SelectArgs a{};
    a.weights = weights_dev, a.num_slots = num_slots, a.num_heads = num_slots ? num_heads : 0, a.slots = slots_dev;
    a.first = first, a.last = last, a.positions = positions_dev, a.out_slots = out_slots_dev, a.shifts = shifts_dev;
    uint32_t* at = (uint32_t*)workspace_dev;
    long long begin = 0, out = 0, keys = 0;
    int n = 0, runs = 0;
    for (int32_t i = 0; i <= n_blocks; ++i) {
      const bool whole = i == n_blocks || n == va::kSelectBlocks;
      if (whole) {
        a.keys = at, a.found = at + keys, a.before = a.found + 4 * n, a.counts = a.before + 2 * runs + (-2 * runs & 3);
        const int rc = va::launch_select_batch(a, n, !large, (hipStream_t)stream);
        if (rc) return rc;
        if (large) at = a.counts + (long long)runs * va::kSelectCounts;
        n = runs = 0, keys = 0;
      }
      if (i == n_blocks) break;
      const long long count = counts_host[i];
      if ((count > va::kSelectInLds) == (large != 0) && keep_host[i] > 0) {
        const int r = large ? (int)va::runs_of(count) : 0;
        a.blocks[n++] = va::SelectBlock{begin, out, count, keep_host[i], keys, r, runs, large ? va::run_tokens_of(count) : 0};
        runs += r;
        if (large) keys += (count + 3) / 4 * 4;
      }
      begin += count, out += keep_host[i];
    }
  }
  return VA_OK;
}
