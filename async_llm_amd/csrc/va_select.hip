// What stays of blocks of tokens: the first and the last few of a block, and of the others the heaviest.
//
//   score(t) = fp32(sum over kv heads, in 64 bits, of weights[h][slots[t]])
//   kept     = the `keep` largest by (protected, score, -t), in rising order of t
//
// Scores become 32-bit keys whose order as whole numbers is theirs (protected tokens above all, NaN next); the keep-th largest key
// is found digit by digit from histograms, most significant first, and then every token above it stays, and of those equal to
// it the first that are wanted.  No sort, and no order of execution that the result depends on.
//
// Blocks of up to kSelectInLds tokens: a workgroup each, keys in LDS, one launch (1500 tokens of 8 heads: 16.1 us).  Longer ones:
// the keys are made by many workgroups, then one per block finds the key at which its list ends and where each run of tokens
// writes, then many write (8 blocks of 60000 .. 131072 tokens: 133 us).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "va_device.h"
#include "va_internal.h"
#include "va_launch.h"

namespace va {

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / kWave;
constexpr int kSelectInLds = 16384;  // tokens of a block whose keys stay in LDS
constexpr int kSelectBlocks = 64;    // blocks of a launch
constexpr int kSelectRun = 4096;     // tokens of a workgroup that makes keys or writes
constexpr int kSelectBins = 256;

struct SelectBlock {
  long long begin, out;  // first entry of its slots, of its results
  long long count, keep;
  long long keys;  // long blocks: first key in the workspace
  int runs, first_run;  // long blocks: runs of kSelectRun tokens; number of the first one in the workspace
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
  uint32_t* keys;    // long blocks
  uint32_t* cut;     // [block][2]: the last key that stays, how many of those equal to it do
  uint32_t* starts;  // [run][2]: kept tokens, tokens equal to the last key in front of a run
  SelectBlock blocks[kSelectBlocks];
};

__device__ __forceinline__ uint32_t select_key(const SelectArgs& a, const SelectBlock& b, long long t) {
  if (t < a.first || t >= b.count - a.last) return 0xffffffffu;
  const long long slot = a.slots[b.begin + t];
  double sum = 0.0;
  if (slot >= 0 && slot < a.num_slots) {
    const float* w = a.weights + slot;
#pragma unroll 8
    for (int h = 0; h < a.num_heads; ++h) sum += (double)w[h * a.num_slots];
  }
  const float score = (float)sum;
  if (score != score) return 0xfffffffeu;
  const uint32_t bits = __float_as_uint(score + 0.f);  // (-0 counts as 0)
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// The keep-th largest of `count` keys and how many of the keys equal to it are among the first `keep`; 1 <= keep <= count.
// All threads of the workgroup call it and get the same.
struct Cut {
  uint32_t key, equal;
};
template <typename Keys>
__device__ __forceinline__ Cut find_cut(Keys key_at, long long count, long long keep, uint32_t (&bins)[kSelectBins], uint32_t (&found)[2]) {
  uint32_t prefix = 0, wanted = (uint32_t)keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < kSelectBins; i += kSelectThreads) bins[i] = 0;
    __syncthreads();
    for (long long t = threadIdx.x; t < count; t += kSelectThreads) {
      const uint32_t key = key_at(t);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&bins[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (threadIdx.x < kWave) {  // lane l: bins 4 l .. + 3; the digit is where the count from above reaches `wanted`
      const int lane = threadIdx.x;
      uint32_t n[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += n[i] = bins[4 * lane + i];
      uint32_t above = sum;  // of this lane's bins and all higher ones
#pragma unroll
      for (int off = 1; off < kWave; off <<= 1) {
        const uint32_t other = __shfl_down(above, off, kWave);
        if (lane + off < kWave) above += other;
      }
      uint32_t higher = above - sum;
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        if (higher < wanted && higher + n[i] >= wanted) found[0] = 4 * lane + i, found[1] = wanted - higher;
        higher += n[i];
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    wanted = found[1];
  }
  return Cut{prefix, wanted};
}

__device__ __forceinline__ uint32_t bits_below(unsigned long long mask, int lane) { return (uint32_t)__popcll(mask & ((1ull << lane) - 1)); }

// A wave's walk over tokens [begin, end) of a block: `write` (or only count) those that stay.  `taken`: kept tokens in front of it,
// `equal`: tokens equal to the cut's key in front of it.
template <bool kWrite, typename Keys>
__device__ __forceinline__ void walk_kept(const SelectArgs& a, const SelectBlock& b, Keys key_at, Cut cut, long long begin, long long end,
                                          uint32_t& taken, uint32_t& equal) {
  const int lane = threadIdx.x % kWave;
  for (long long t0 = begin; t0 < end; t0 += kWave) {
    const long long t = t0 + lane;
    const uint32_t key = t < end ? key_at(t) : 0u;
    const bool same = t < end && key == cut.key;
    const unsigned long long sames = __ballot(same);
    const bool stays = t < end && (key > cut.key || (same && equal + bits_below(sames, lane) < cut.equal));
    const unsigned long long kept = __ballot(stays);
    if (kWrite && stays) {
      const long long rank = (long long)taken + bits_below(kept, lane), at = b.out + rank;
      a.positions[at] = t;
      a.out_slots[at] = a.slots[b.begin + t];
      a.shifts[at] = rank - t;
    }
    equal += (uint32_t)__popcll(sames);
    taken += (uint32_t)__popcll(kept);
  }
}

__global__ __launch_bounds__(kSelectThreads) void select_kernel(SelectArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t bins[kSelectBins], found[2], of_wave[kSelectWaves][2];
  const SelectBlock& b = a.blocks[blockIdx.x];
  if (b.keep == 0) return;
  const int count = (int)b.count;
  for (int t = threadIdx.x; t < count; t += kSelectThreads) keys[t] = select_key(a, b, t);
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
  uint32_t taken = above + min(same, cut.equal);
  walk_kept<true>(a, b, key_at, cut, begin, end, taken, same);
}

// ---- long blocks ----
__global__ __launch_bounds__(kSelectThreads) void select_keys_kernel(SelectArgs a) {
  const SelectBlock& b = a.blocks[blockIdx.y];
  if ((int)blockIdx.x >= b.runs) return;
  const long long begin = (long long)blockIdx.x * kSelectRun, end = min(begin + kSelectRun, b.count);
  for (long long t = begin + threadIdx.x; t < end; t += kSelectThreads) a.keys[b.keys + t] = select_key(a, b, t);
}

__global__ __launch_bounds__(kSelectThreads) void select_cut_kernel(SelectArgs a) {
  __shared__ uint32_t bins[kSelectBins], found[2];
  const SelectBlock& b = a.blocks[blockIdx.x];
  if (b.keep == 0) return;
  const uint32_t* keys = a.keys + b.keys;
  auto key_at = [&](long long t) __attribute__((always_inline)) { return keys[t]; };
  const Cut cut = find_cut(key_at, b.count, b.keep, bins, found);
  if (threadIdx.x == 0) a.cut[2 * blockIdx.x] = cut.key, a.cut[2 * blockIdx.x + 1] = cut.equal;
  // counts of the runs, a wave each
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  for (int run = wave; run < b.runs; run += kSelectWaves) {
    const long long begin = (long long)run * kSelectRun, end = min(begin + kSelectRun, b.count);
    uint32_t above = 0, same = 0;
    for (long long t = begin + lane; t < end; t += kWave) above += keys[t] > cut.key, same += keys[t] == cut.key;
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) above += __shfl_xor(above, off, kWave), same += __shfl_xor(same, off, kWave);
    if (lane == 0) a.starts[2 * (b.first_run + run)] = above, a.starts[2 * (b.first_run + run) + 1] = same;
  }
}

__global__ __launch_bounds__(kSelectThreads) void select_write_kernel(SelectArgs a) {
  __shared__ uint32_t of_wave[kSelectWaves][2];
  const SelectBlock& b = a.blocks[blockIdx.y];
  if ((int)blockIdx.x >= b.runs || b.keep == 0) return;
  const uint32_t* keys = a.keys + b.keys;
  const Cut cut{a.cut[2 * blockIdx.y], a.cut[2 * blockIdx.y + 1]};
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  // what stays in front of this run, and of this wave's part of it
  uint32_t above = 0, same = 0;
  for (int run = lane; run < (int)blockIdx.x; run += kWave) above += a.starts[2 * (b.first_run + run)], same += a.starts[2 * (b.first_run + run) + 1];
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) above += __shfl_xor(above, off, kWave), same += __shfl_xor(same, off, kWave);
  constexpr int kEach = kSelectRun / kSelectWaves;
  const long long begin = min((long long)blockIdx.x * kSelectRun + wave * kEach, b.count), end = min(begin + kEach, b.count);
  uint32_t own_above = 0, own_same = 0;
  for (long long t = begin + lane; t < end; t += kWave) own_above += keys[t] > cut.key, own_same += keys[t] == cut.key;
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) own_above += __shfl_xor(own_above, off, kWave), own_same += __shfl_xor(own_same, off, kWave);
  if (lane == 0) of_wave[wave][0] = own_above, of_wave[wave][1] = own_same;
  __syncthreads();
  for (int w = 0; w < wave; ++w) above += of_wave[w][0], same += of_wave[w][1];
  uint32_t taken = above + min(same, cut.equal);
  walk_kept<true>(a, b, [&](long long t) __attribute__((always_inline)) { return keys[t]; }, cut, begin, end, taken, same);
}

static long long runs_of(long long count) { return (count + kSelectRun - 1) / kSelectRun; }

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
    hipLaunchKernelGGL(select_keys_kernel, dim3((unsigned)runs, (unsigned)n), block, 0, stream, a);
    hipLaunchKernelGGL(select_cut_kernel, dim3((unsigned)n), block, 0, stream, a);
    hipLaunchKernelGGL(select_write_kernel, dim3((unsigned)runs, (unsigned)n), block, 0, stream, a);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VA_OK : va_fail(VA_ERR_HIP, "selection launch: %s", hipGetErrorString(e));
}

// Words of the workspace: keys, cuts, starts of the runs of all long blocks (batches start on 16-byte boundaries); -1 for counts that no selection takes.
static int64_t select_words(int32_t n_blocks, const int64_t* counts) {
  int64_t words = 0;
  for (int32_t i = 0; i < n_blocks; ++i) {
    if (counts[i] < 0 || counts[i] > 0x7fffffffLL) return -1;
    if (counts[i] > kSelectInLds) words += (counts[i] + 3) / 4 * 4 + 4 + 2 * runs_of(counts[i]);
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
        a.keys = at, a.cut = at + keys, a.starts = a.cut + 2 * n;
        const int rc = va::launch_select_batch(a, n, !large, (hipStream_t)stream);
        if (rc) return rc;
        if (large) at = a.starts + 2 * runs + (-(2 * n + 2 * runs) & 3);
        n = runs = 0, keys = 0;
      }
      if (i == n_blocks) break;
      const long long count = counts_host[i];
      if ((count > va::kSelectInLds) == (large != 0) && keep_host[i] > 0) {
        const int r = large ? (int)va::runs_of(count) : 0;
        a.blocks[n++] = va::SelectBlock{begin, out, count, keep_host[i], keys, r, runs};
        runs += r;
        if (large) keys += (count + 3) / 4 * 4;
      }
      begin += count, out += keep_host[i];
    }
  }
  return VA_OK;
}
