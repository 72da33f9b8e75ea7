// The tables of a packed batch (sequences one after the other on one token
// axis), built on the GPU from the sequences' lengths: no length is copied to
// the host, so a batch may be planned inside a captured graph.
//
//   cu [N + 2]     first row of every sequence; cu[N] ends the last one, and
//                  rows cu[N] .. cu[N + 1] = T are padding ("sequence" N)
//   pos [T]        position of a row inside its sequence, -1 for padding
//   seq [T]        its sequence, -1 for padding
//   jobs [J] int4  (first row, rows, block of 128 rows, keys) of a sequence's
//                  blocks (keys = rows, 0 for the padding), longest sweep
//                  first: a causal query block b sweeps b + 1 key blocks, and
//                  its mirror image (the key block nblk - 1 - b) is swept by
//                  as many query blocks, so one table orders forward and
//                  backward.  All a workgroup needs is in its slot: one load,
//                  not a chain of two.  Slots past the last job hold rows = 0.
//
// Two launches, once per batch: 6 to 8 us for the jobs (one workgroup: scans,
// a counting sort by sweep length) and 2 to 3 us for the rows' tables; the
// layers of a model share them.
//
// Lengths below zero count as zero, and what passes T is cut off, so no table
// entry ever points outside the batch's rows.
#include "common.h"

using namespace kgwe;

namespace {

constexpr int kBlock = 128;     // rows of a job, as in packed_attn.hip
constexpr int kThreads = 1024;  // the one workgroup of the job kernel
constexpr int kBuckets = 2048;  // sweep lengths told apart by the job order

// Exclusive prefix sum of one value per thread over the workgroup; *total gets
// the sum.  Two barriers; `sh` holds one value per wave.
__device__ __forceinline__ int block_scan(int v, int* sh, int* total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int x = v;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int y = __shfl_up(x, off, kWave);
    if (lane >= off) x += y;
  }
  __syncthreads();  // sh of the previous call has been read
  if (lane == kWave - 1) sh[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kThreads / kWave; ++w) {
    if (w < wave) before += sh[w];
    all += sh[w];
  }
  *total = all;
  return before + x - v;
}

// Largest i in [0, n) with a[i] <= x; a[0] <= x.
__device__ __forceinline__ int last_at_most(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// first [N + 2]: workspace, the number of each sequence's first job.
__global__ __launch_bounds__(kThreads) void plan_kernel(const int* __restrict__ lengths, int N, int T, int* cu,
                                                        int* first, int4* __restrict__ jobs, int J) {
  __shared__ int sh[kThreads / kWave];
  __shared__ int count[kBuckets];
  // 1. rows: running sum of the lengths, cut at T
  int base = 0;
  for (int i0 = 0; i0 < N; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    const int len = i < N ? min(max(lengths[i], 0), T) : 0;
    // The running sum may pass 2^31 long before the cut: saturate.
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    long long x = len;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const long long y = __shfl_up(x, off, kWave);
      if (lane >= off) x += y;
    }
    __syncthreads();
    if (lane == kWave - 1) sh[wave] = static_cast<int>(min(x, static_cast<long long>(T)));
    __syncthreads();
    long long before = 0, all = 0;
    for (int w = 0; w < kThreads / kWave; ++w) {
      if (w < wave) before += sh[w];
      all += sh[w];
    }
    if (i < N) cu[i] = static_cast<int>(min(base + before + x - len, static_cast<long long>(T)));
    base = static_cast<int>(min(base + all, static_cast<long long>(T)));
  }
  if (threadIdx.x == 0) {
    cu[N] = base;
    cu[N + 1] = T;
  }
  __syncthreads();  // one workgroup: its own global writes are visible to it after the barrier
  // 2. jobs: running sum of the block counts (the padding counts as sequence N)
  int njobs = 0;
  for (int i0 = 0; i0 <= N; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    const int nb = i <= N ? (cu[i + 1] - cu[i] + kBlock - 1) / kBlock : 0;
    int all;
    const int x = block_scan(nb, sh, &all);
    if (i <= N) first[i] = njobs + x;
    njobs += all;
  }
  if (threadIdx.x == 0) first[N + 1] = njobs;
  for (int b = threadIdx.x; b < kBuckets; b += kThreads) count[b] = 0;
  __syncthreads();
  njobs = min(njobs, J);
  // 3. order by sweep length, longest first (padding last): counting sort.  The
  // order inside a bucket is whatever the atomics give; no result depends on it.
  auto bucket = [&](int s, int b) { return s == N ? kBuckets - 1 : kBuckets - 2 - min(b, kBuckets - 2); };
  for (int j = threadIdx.x; j < njobs; j += kThreads) {
    const int s = last_at_most(first, N + 1, j);
    atomicAdd(&count[bucket(s, j - first[s])], 1);
  }
  __syncthreads();
  {
    int all;
    const int c0 = count[2 * threadIdx.x], c1 = count[2 * threadIdx.x + 1];
    const int x = block_scan(c0 + c1, sh, &all);
    __syncthreads();
    count[2 * threadIdx.x] = x;
    count[2 * threadIdx.x + 1] = x + c0;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < njobs; j += kThreads) {
    const int s = last_at_most(first, N + 1, j);
    const int b = j - first[s];
    const int row0 = cu[s], rows = cu[s + 1] - row0;
    jobs[atomicAdd(&count[bucket(s, b)], 1)] = make_int4(row0, rows, b, s < N ? rows : 0);
  }
  for (int j = njobs + threadIdx.x; j < J; j += kThreads) jobs[j] = make_int4(0, 0, 0, 0);
}
static_assert(kBuckets == 2 * kThreads, "two buckets per thread");

__global__ __launch_bounds__(256) void rows_kernel(const int* __restrict__ cu, int N, int T,
                                                   int* __restrict__ pos, int* __restrict__ seq) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= T) return;
  const int s = last_at_most(cu, N + 1, t);
  pos[t] = s < N ? t - cu[s] : -1;
  seq[t] = s < N ? s : -1;
}

}  // namespace

// Job slots that a batch of N sequences on T rows can need.
KGWE_API int kgwe_packed_plan_jobs(int N, int T) {
  if (N < 0 || T <= 0) return 0;
  const int64_t most = static_cast<int64_t>(T) / kBlock + N + 1;
  return static_cast<int>(most < T ? most : T);
}

// cu and first: int32 [N + 2]; jobs: int32 [jobs, 4], 16-byte aligned; pos, seq: int32 [T].
KGWE_API int kgwe_packed_plan(const int* lengths, int N, int T, int* cu, int* first, int* jobs, int J, int* pos,
                              int* seq, hipStream_t s) {
  if (N < 0 || T <= 0 || J < kgwe_packed_plan_jobs(N, T) || N > (1 << 24) || T > 0x7fffffff - 256) return -1;
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kThreads), 0, s, lengths, N, T, cu, first,
                     reinterpret_cast<int4*>(jobs), J);
  if (int rc = KGWE_CHECK_LAUNCH()) return rc;
  hipLaunchKernelGGL(rows_kernel, dim3((T + 255) / 256), dim3(256), 0, s, cu, N, T, pos, seq);
  return KGWE_CHECK_LAUNCH();
}
