// layer_norm.cu -- layer norm over the last dimension of a rank 1-3 view.
//
//   mean = sum x / N,  var = sum (x - mean)^2 / N,  rstd = 1 / sqrt(var + eps)
//   xh = (x - mean) rstd,  y = xh w + b
// Sums are held in f32; x, w and b are widened exactly, y is rounded once to
// its type.  A few operations an element: bound by memory.  A row's elements
// stay on the SM, so that the variance is taken around the mean from the same
// read.
#include "layer_norm.cuh"

namespace cg = cooperative_groups;

namespace spmdb200 {

namespace {

constexpr int kMost = 16;         // elements of a row in a thread
constexpr int kHalfLanes = 512;   // threads of a block for rows past kThreads * kMost columns
constexpr int kLongLanes = 1024;  // threads of a block for long rows of any strides,
constexpr int kCluster = 8;       // and at most so many of them share a row
constexpr int64_t kHeld = (int64_t)kThreads * kMost, kHalfHeld = (int64_t)kHalfLanes * kMost;
constexpr int64_t kLongRun = (int64_t)kLongLanes * kMost;

// Streamed rows (layer_norm.cuh): weight and bias are loaded once a thread.  A
// group of lanes takes R rows at a time, one or two: the two reductions of a row
// are a long chain of waits, and a second row fills them where rows are 16-bit (101
// against 121 us for 32768 x 4096; f32 rows wait for memory, and are faster with one
// at a time and a stage more: 124 against 141 us).
template <int MAXT>
constexpr int kStages = MAXT > kThreads ? 2 : 3;

template <class TX, class TY, int W, int NV, int R, int MAXT, bool WRAPS, bool APART>
__global__ void __launch_bounds__(MAXT, MAXT > kThreads ? 1 : NV * W * R > 8 ? 2 : 3)
ln_forward_stream(const TX *x, const __grid_constant__ RowWalk xr, TY *y, const __grid_constant__ RowWalk yr, const void *w,
                  const void *b, int wtype, int64_t rows, int cols, float eps, float *mean_out, float *rstd_out, int lanes) {
  using In = Source<W, NV, MAXT, APART, TX>;
  constexpr int kStage = R * In::kBytes;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(16) F2 sh[2][32];
  const int lane = threadIdx.x & (lanes - 1), groups = MAXT / lanes, group = threadIdx.x / lanes;
  const float inv_n = 1.0f / (float)cols;
  const int64_t step = (int64_t)gridDim.x * groups, i = (int64_t)blockIdx.x * groups + group;
  const int mine = row_count(i, rows, step), turns = row_count(i - group, rows, step);
  const TX *from = x + (mine ? row_offset(xr.r, i) : 0);
  TY *to = y + (mine ? row_offset(yr.r, i) : 0);
  const int shift = (int)((APART ? (uintptr_t)to / sizeof(TY) : (uintptr_t)from / sizeof(TX)) % W);
  const Held<W, NV> have = held<W, NV>(cols, lane, lanes, shift);
  In in;
  in.place(from, cols, lane, lanes, shift, have, smem, kStages<MAXT> * R, In::kBytes);
  to += lane * W - shift;
  from += in.start;
  int stage_in = 0, stage = 0, fetched = 0;  // stages as offsets
  auto fetch = [&] {
    In::emptied();
#pragma unroll
    for (int q = 0; q < R; ++q) {
      if (fetched < mine) in.fetch(stage_in + q * In::kBytes, from);
      ++fetched;
      from = next_row<WRAPS>(from, x + in.start, xr, i + fetched * step);
    }
    copy_commit();  // empty past the last row, so that the count of groups stays
    stage_in = stage_in == (kStages<MAXT> - 1) * kStage ? 0 : stage_in + kStage;
  };
#pragma unroll
  for (int q = 0; q < kStages<MAXT> - 1; ++q) fetch();
  float wv[NV][W], bv[NV][W];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_weight<W, true>(w, wtype, 0, 0, cols, k, lane, lanes, shift, 1.0f, wv[k]);
    load_weight<W, true>(b, wtype, 0, 0, cols, k, lane, lanes, shift, 0.0f, bv[k]);
  }
  // R sums of a row each, as a pair.
  auto sums = [&](const F2 (&t)[R], int space) {
    if constexpr (R == 2) return row_sum2<MAXT>({t[0].x + t[0].y, t[1].x + t[1].y}, lanes, sh[space]);
    else return both(row_sum(t[0].x + t[0].y, lanes, &sh[space]->x));
  };
  for (int turn = 0; turn < turns; turn += R) {
    fetch();
    copy_wait<kStages<MAXT> - 1>();
    F2 v[R][NV][W / 2], t[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      in.arrived(stage + q * In::kBytes);
      t[q] = {0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        in.take(stage + q * In::kBytes, k, v[q][k]);
#pragma unroll
        for (int e = 0; e < W / 2; ++e) t[q] = add2(t[q], v[q][k][e]);
      }
    }
    stage = stage == (kStages<MAXT> - 1) * kStage ? 0 : stage + kStage;
    const F2 mean2 = mul2(sums(t, 0), both(inv_n));
#pragma unroll
    for (int q = 0; q < R; ++q) {
      t[q] = deviations<W, NV>(v[q], q ? mean2.y : mean2.x, have);
    }
    const F2 var2 = mul2(sums(t, 1), both(inv_n));
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const float rstd = 1.0f / sqrtf((q ? var2.y : var2.x) + eps);
      if (turn + q < mine) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int e = 0; e < W / 2; ++e)
            v[q][k][e] = fma2(mul2(v[q][k][e], both(rstd)), {wv[k][2 * e], wv[k][2 * e + 1]}, {bv[k][2 * e], bv[k][2 * e + 1]});
        stream_store<W, NV>(to, have, lanes, v[q]);
        if (lane == 0) {
          if (mean_out) mean_out[i + (turn + q) * step] = q ? mean2.y : mean2.x;
          if (rstd_out) rstd_out[i + (turn + q) * step] = rstd;
        }
      }
      to = next_row<WRAPS>(to, y + lane * W - shift, yr, i + (turn + q + 1) * step);
    }
  }
  copy_wait<0>();
}

// Longer rows that a cluster's blocks hold, several at a time.  One exchange gives
// both statistics: each warp's sum, and its squares around its own mean (8192 x
// 16384 f32: 208 us, with two exchanges as above 239).  An exchange costs the more
// the fewer bytes are under way: 16-bit rows go four at a time (148 us, two 174).
// As many clusters as are resident, whatever rows they take where all start
// alike: 201 and 136 us, 5.3 and 3.9 TB/s; what is left is the exchange's wait.
template <class TX>
constexpr int kSpreadRows = 8 / (int)sizeof(TX);
template <class TX, bool APART>
constexpr int kSpreadStages = APART && sizeof(TX) == 2 ? 2 : 3;  // as two blocks' stages and sums fit an SM

template <class TX, class TY, int W, bool WRAPS, bool APART>
__global__ void __launch_bounds__(kThreads, 2)
ln_forward_spread(const TX *x, const __grid_constant__ RowWalk xr, TY *y, const __grid_constant__ RowWalk yr, const void *w,
                  const void *b, int wtype, int64_t rows, int cols, float eps, float *mean_out, float *rstd_out, int blocks) {
  constexpr int NV = kMost / W, R = kSpreadRows<TX>, kWarps = kThreads / 32, kStages = kSpreadStages<TX, APART>;
  using In = Source<W, NV, kThreads, APART, TX>;
  constexpr int kStage = R * In::kBytes;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(16) float4 sh[2][R / 2][kSpread * kWarps];
  __shared__ float2 count[kSpread * kWarps];  // a warp's columns of a row, and their reciprocal
  cluster_arrive();
  const int rank = blockIdx.x % blocks, lanes = blocks * kThreads, lane = rank * kThreads + threadIdx.x, entry = lane >> 5;
  const float inv_n = 1.0f / (float)cols;
  const int64_t step = gridDim.x / blocks, i = blockIdx.x / blocks;
  const int turns = row_count(i, rows, step);
  const TX *from = x + row_offset(xr.r, i);
  TY *to = y + row_offset(yr.r, i);
  const int shift = (int)((APART ? (uintptr_t)to / sizeof(TY) : (uintptr_t)from / sizeof(TX)) % W);
  const Held<W, NV> have = held<W, NV>(cols, lane, lanes, shift);
  In in;
  in.place(from, cols, lane, lanes, shift, have, smem, kStages * R, In::kBytes);
  to += lane * W - shift;
  from += in.start;
  int stage_in = 0, stage = 0, fetched = 0;
  auto fetch = [&] {
    In::emptied();
#pragma unroll
    for (int q = 0; q < R; ++q) {
      if (fetched < turns) in.fetch(stage_in + q * In::kBytes, from);
      ++fetched;
      from = next_row<WRAPS>(from, x + in.start, xr, i + fetched * step);
    }
    copy_commit();  // empty past the last row, so that the count of groups stays
    stage_in = stage_in == (kStages - 1) * kStage ? 0 : stage_in + kStage;
  };
#pragma unroll
  for (int q = 0; q < kStages - 1; ++q) fetch();
  for (int e = threadIdx.x; e < blocks * kWarps; e += kThreads) {  // as held() has it
    int n = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int low = (k * lanes + 32 * e) * W - shift, high = low + 32 * W;
      n += max(min(high, cols) - max(low, 0), 0);
    }
    count[e] = make_float2((float)n, n ? 1.0f / (float)n : 0.0f);
  }
  __syncthreads();
  const float own = count[entry].y;
  float wv[NV][W], bv[NV][W];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_weight<W, true>(w, wtype, 0, 0, cols, k, lane, lanes, shift, 1.0f, wv[k]);
    load_weight<W, true>(b, wtype, 0, 0, cols, k, lane, lanes, shift, 0.0f, bv[k]);
  }
  cluster_wait();  // the others have begun
  for (int turn = 0, space = 0; turn < turns; turn += R, space ^= 1) {
    fetch();
    copy_wait<kStages - 1>();
    F2 t[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      in.arrived(stage + q * In::kBytes);
      t[q] = {0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        F2 v[W / 2];
        in.take(stage + q * In::kBytes, k, v);
#pragma unroll
        for (int e = 0; e < W / 2; ++e) t[q] = add2(t[q], v[e]);
      }
    }
    F2 sum[R / 2], mean[R / 2], var[R / 2];  // of two rows each
#pragma unroll
    for (int p = 0; p < R / 2; ++p) sum[p] = row_sum2<kThreads>({t[2 * p].x + t[2 * p].y, t[2 * p + 1].x + t[2 * p + 1].y}, 32, nullptr);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      F2 v[NV][W / 2];
#pragma unroll
      for (int k = 0; k < NV; ++k) in.take(stage + q * In::kBytes, k, v[k]);
      t[q] = deviations<W, NV>(v, (q & 1 ? sum[q / 2].y : sum[q / 2].x) * own, have);
    }
#pragma unroll
    for (int p = 0; p < R / 2; ++p)
      cluster_share({sum[p], row_sum2<kThreads>({t[2 * p].x + t[2 * p].y, t[2 * p + 1].x + t[2 * p + 1].y}, 32, nullptr)}, blocks, entry,
                    sh[space][p]);
    cluster_arrive();
    cluster_wait();
#pragma unroll
    for (int p = 0; p < R / 2; ++p) {
      const float4 *shared = sh[space][p];
      mean[p] = var[p] = {0.0f, 0.0f};
      for (int e = threadIdx.x & 31; e < blocks * kWarps; e += 32) mean[p] = add2(mean[p], {shared[e].x, shared[e].y});
      mean[p] = mul2(row_sum2<kThreads>(mean[p], 32, nullptr), both(inv_n));
      for (int e = threadIdx.x & 31; e < blocks * kWarps; e += 32) {
        const float4 s = shared[e];
        const float2 n = count[e];
        const F2 d = fma2({s.x, s.y}, both(n.y), {-mean[p].x, -mean[p].y});
        var[p] = add2(var[p], fma2(mul2(d, both(n.x)), d, {s.z, s.w}));
      }
      var[p] = mul2(row_sum2<kThreads>(var[p], 32, nullptr), both(inv_n));
    }
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const float m = q & 1 ? mean[q / 2].y : mean[q / 2].x, rstd = 1.0f / sqrtf((q & 1 ? var[q / 2].y : var[q / 2].x) + eps);
      if (turn + q < turns) {
        F2 v[NV][W / 2];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          in.take(stage + q * In::kBytes, k, v[k]);
#pragma unroll
          for (int e = 0; e < W / 2; ++e)
            v[k][e] = fma2(mul2(add2(v[k][e], both(-m)), both(rstd)), {wv[k][2 * e], wv[k][2 * e + 1]}, {bv[k][2 * e], bv[k][2 * e + 1]});
        }
        stream_store<W, NV>(to, have, lanes, v);
        if (lane == 0) {
          if (mean_out) mean_out[i + (turn + q) * step] = m;
          if (rstd_out) rstd_out[i + (turn + q) * step] = rstd;
        }
      }
      to = next_row<WRAPS>(to, y + lane * W - shift, yr, i + (turn + q + 1) * step);
    }
    stage = stage == (kStages - 1) * kStage ? 0 : stage + kStage;
  }
  copy_wait<0>();
}

// Rows of any strides.  Rows past the last take part in the barriers, with no
// columns.
template <class TX, class TY, int W, int NV>
__global__ void __launch_bounds__(kThreads, 3)
ln_forward(const TX *x, Rows xr, TY *y, Rows yr, const void *w, const void *b, int wtype, int64_t rows, int cols, float eps,
           float *mean_out, float *rstd_out, int lanes) {
  __shared__ float sh[2][32];
  const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes;
  const float inv_n = 1.0f / (float)cols;
  const int64_t step = (int64_t)gridDim.x * (kThreads / lanes);
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / lanes) + group; i - group < rows; i += step) {
    const int n = i < rows ? cols : 0;
    float v[NV][W], s = 0.0f;
    load_row<W, NV>(x + (n ? row_offset(xr, i) : 0), xr.sc, n, lane, lanes, 0.0f, v);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < W; ++e) s += v[k][e];
    const float mean = row_sum(s, lanes, sh[0]) * inv_n;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < W; ++e) {
        v[k][e] -= mean;
        if (column<W, false>(k, e, lane, lanes, 0) < n) s = fmaf(v[k][e], v[k][e], s);
      }
    const float rstd = 1.0f / sqrtf(row_sum(s, lanes, sh[1]) * inv_n + eps);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float wv[W], bv[W];
      load_weight<W, false>(w, wtype, 0, 0, n, k, lane, lanes, 0, 1.0f, wv);
      load_weight<W, false>(b, wtype, 0, 0, n, k, lane, lanes, 0, 0.0f, bv);
#pragma unroll
      for (int e = 0; e < W; ++e) v[k][e] = fmaf(v[k][e] * rstd, wv[e], bv[e]);
    }
    store_row<W, NV>(y + (n ? row_offset(yr, i) : 0), yr.sc, n, lane, lanes, v);
    if (lane == 0 && n) {
      if (mean_out) mean_out[i] = mean;
      if (rstd_out) rstd_out[i] = rstd;
    }
  }
}

// Two sets' count, mean and sum of squares around it join into those of both.  An
// empty set's d is the other's whole mean, whose square may leave f32: the product
// begins with the counts, which are zero then.
struct Moments {
  float n, mean, m2;
};
__device__ __forceinline__ Moments join(Moments a, Moments b) {
  const float n = a.n + b.n;
  if (n == 0.0f) return a;
  const float d = b.mean - a.mean, share = b.n / n;
  return {n, fmaf(d, share, a.mean), a.m2 + b.m2 + d * (d * (a.n * share))};
}
__device__ __forceinline__ Moments join_warp(Moments a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = join(a, {__shfl_xor_sync(0xffffffffu, a.n, o), __shfl_xor_sync(0xffffffffu, a.mean, o),
                 __shfl_xor_sync(0xffffffffu, a.m2, o)});
  return {__shfl_sync(0xffffffffu, a.n, 0), __shfl_sync(0xffffffffu, a.mean, 0), __shfl_sync(0xffffffffu, a.m2, 0)};
}

// Longer rows, first pass: moments of each run of a row.
constexpr int kCutStages = 4;

template <class TX, int W, bool WRAPS>
__global__ void __launch_bounds__(kThreads, 4)
ln_moments(const TX *x, const __grid_constant__ RowWalk xr, int64_t cols, const __grid_constant__ Cut cut, float4 *shares) {
  constexpr int NV = kCutMost / W;
  using In = Source<W, NV, kThreads, false, TX>;
  constexpr int kStage = In::kBytes;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Moments warps[kCutRows][kCutWarps];
  const CutPlace at = cut_place(cut);
  pdl_trigger();
  if (at.rows == 0) return pdl_wait();
  const int lane = threadIdx.x;
  const TX *from = x + row_offset(xr.r, at.i);
  const int64_t first = at.run * kRun;
  const int start = (int)((uintptr_t)from / sizeof(TX) % W);
  // The run's columns, relative to `first`: from `low` (0 or the run before's end) to `high`.
  const int low = at.run == 0 ? 0 : -start, high = cols - first < kRun - start ? (int)(cols - first) : kRun - start;
  // As a row of its own that starts `shift` elements into its first vector.
  const int shift = at.run == 0 ? start : 0, n = high - low;
  const Held<W, NV> have = held<W, NV>(n, lane, kThreads, shift);
  In in;
  in.place(from + first + low, n, lane, kThreads, shift, have, smem, kCutStages, kStage);
  from += first + low + in.start;
  float count = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) count += (float)__popc(have.in[k]);
  const float inv_count = count > 0.0f ? 1.0f / count : 0.0f, all = warp_sum_f32(count), inv_all = all > 0.0f ? 1.0f / all : 0.0f;
  int stage_in = 0, stage = 0, fetched = 0;
  auto fetch = [&] {
    In::emptied();
    if (fetched < at.rows) in.fetch(stage_in, from);
    copy_commit();
    ++fetched;
    from = next_row<WRAPS>(from, x + first + low + in.start, xr, at.i + (int64_t)fetched * cut.parts);
    stage_in = stage_in == (kCutStages - 1) * kStage ? 0 : stage_in + kStage;
  };
#pragma unroll
  for (int q = 0; q < kCutStages - 1; ++q) fetch();
  for (int turn = 0; turn < at.rows; ++turn) {
    fetch();
    copy_wait<kCutStages - 1>();
    in.arrived(stage);
    F2 v[NV][W / 2], t{0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      in.take(stage, k, v[k]);
#pragma unroll
      for (int e = 0; e < W / 2; ++e) t = add2(t, v[k][e]);
    }
    stage = stage == (kCutStages - 1) * kStage ? 0 : stage + kStage;
    // Around the thread's mean, then the threads' means around the warp's.
    const float sum = t.x + t.y, mean = sum * inv_count;
    t = deviations<W, NV>(v, mean, have);
    const float warp_mean = warp_sum_f32(sum) * inv_all, d = mean - warp_mean;
    const float m2 = warp_sum_f32(fmaf(count * d, d, t.x + t.y));
    if ((lane & 31) == 0) warps[turn][lane >> 5] = {all, warp_mean, m2};
  }
  copy_wait<0>();
  __syncthreads();
  pdl_wait();  // the shares of the batch before have been read
  if (lane < at.rows) {
    Moments m = warps[lane][0];
#pragma unroll
    for (int k = 1; k < kCutWarps; ++k) m = join(m, warps[lane][k]);
    shares[(at.i - cut.first + (int64_t)lane * cut.parts) * cut.runs + at.run] = make_float4(m.n, m.mean, m.m2, 0.0f);
  }
}

// Second pass: the rows' statistics from the shares, and the output.
template <class TX, class TY, int W, bool WRAPS, bool APART>
__global__ void __launch_bounds__(kThreads, 2)
ln_outputs(const TX *x, const __grid_constant__ RowWalk xr, TY *y, const __grid_constant__ RowWalk yr, const void *w, const void *b,
           int wtype, int64_t cols, float eps, float *mean_out, float *rstd_out, const __grid_constant__ Cut cut, const float4 *shares) {
  constexpr int NV = kCutMost / W;
  using In = Source<W, NV, kThreads, APART, TX>;
  constexpr int kStage = In::kBytes;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float2 stats[kCutRows];  // -mean, rstd
  const CutPlace at = cut_place(cut);
  pdl_trigger();
  if (at.rows == 0) return pdl_wait();
  const int lane = threadIdx.x;
  const TX *from = x + row_offset(xr.r, at.i);
  TY *to = y + row_offset(yr.r, at.i);
  const int64_t first = at.run * kRun;
  const int start = (int)((APART ? (uintptr_t)to / sizeof(TY) : (uintptr_t)from / sizeof(TX)) % W);
  const int low = at.run == 0 ? 0 : -start, high = cols - first < kRun - start ? (int)(cols - first) : kRun - start;
  const int shift = at.run == 0 ? start : 0, n = high - low;
  const Held<W, NV> have = held<W, NV>(n, lane, kThreads, shift);
  In in;
  in.place(from + first + low, n, lane, kThreads, shift, have, smem, kCutStages, kStage);
  to += first + low + lane * W - shift;
  from += first + low + in.start;
  int stage_in = 0, stage = 0, fetched = 0;
  auto fetch = [&] {
    In::emptied();
    if (fetched < at.rows) in.fetch(stage_in, from);
    copy_commit();
    ++fetched;
    from = next_row<WRAPS>(from, x + first + low + in.start, xr, at.i + (int64_t)fetched * cut.parts);
    stage_in = stage_in == (kCutStages - 1) * kStage ? 0 : stage_in + kStage;
  };
#pragma unroll
  for (int q = 0; q < kCutStages - 1; ++q) fetch();
  float wv[NV][W], bv[NV][W];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_weight<W, true>(w, wtype, first + low, 0, n, k, lane, kThreads, shift, 1.0f, wv[k]);
    load_weight<W, true>(b, wtype, first + low, 0, n, k, lane, kThreads, shift, 0.0f, bv[k]);
  }
  pdl_wait();  // the shares are there
  for (int r = lane >> 5; r < at.rows; r += kCutWarps) {  // a warp a row, in one order
    const int64_t i = at.i + (int64_t)r * cut.parts;
    Moments m{0.0f, 0.0f, 0.0f};
    for (int64_t q = lane & 31; q < cut.runs; q += 32) {
      const float4 s = shares[(i - cut.first) * cut.runs + q];
      m = join(m, {s.x, s.y, s.z});
    }
    m = join_warp(m);
    const float rstd = 1.0f / sqrtf(m.m2 / (float)cols + eps);
    if ((lane & 31) == 0) {
      stats[r] = make_float2(-m.mean, rstd);
      if (at.run == 0) {
        if (mean_out) mean_out[i] = m.mean;
        if (rstd_out) rstd_out[i] = rstd;
      }
    }
  }
  __syncthreads();
  for (int turn = 0; turn < at.rows; ++turn) {
    fetch();
    copy_wait<kCutStages - 1>();
    if constexpr (APART) in.arrived(stage);  // elements before a row's start are stored nowhere
    const float2 stat = stats[turn];
    F2 v[NV][W / 2];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      in.take(stage, k, v[k]);
#pragma unroll
      for (int e = 0; e < W / 2; ++e)
        v[k][e] = fma2(mul2(add2(v[k][e], both(stat.x)), both(stat.y)), {wv[k][2 * e], wv[k][2 * e + 1]}, {bv[k][2 * e], bv[k][2 * e + 1]});
    }
    stage = stage == (kCutStages - 1) * kStage ? 0 : stage + kStage;
    stream_store<W, NV>(to, have, kThreads, v);
    to = next_row<WRAPS>(to, y + first + low + lane * W - shift, yr, at.i + (int64_t)(turn + 1) * cut.parts);
  }
  copy_wait<0>();
}

// Longer rows of any strides: a cluster reads them twice, the second time from L2.
// A thread's elements are taken kMost at a time.
template <class TX, class TY, int W>
__global__ void __launch_bounds__(kLongLanes)
ln_forward_long(const TX *x, Rows xr, TY *y, Rows yr, const void *w, const void *b, int wtype, int64_t rows, int64_t cols,
                float eps, float *mean_out, float *rstd_out) {
  constexpr int NV = kMost / W;
  __shared__ Moments sh[kLongLanes / 32], mine;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), lane = threadIdx.x & 31;
  const int64_t runs = (cols + kLongRun - 1) / kLongRun;
  for (int64_t i = blockIdx.x / blocks; i < rows; i += gridDim.x / blocks) {
    const TX *px = x + row_offset(xr, i);
    TY *py = y + row_offset(yr, i);
    Moments m{0.0f, 0.0f, 0.0f};
    float v[NV][W];
    for (int64_t r = rank; r < runs; r += blocks) {
      const int n = cols - r * kLongRun < kLongRun ? (int)(cols - r * kLongRun) : (int)kLongRun;
      load_row<W, NV>(px + r * kLongRun * xr.sc, xr.sc, n, threadIdx.x, kLongLanes, 0.0f, v);
      Moments t{0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < W; ++e) {
          t.mean += v[k][e];
          t.n += column<W, false>(k, e, threadIdx.x, kLongLanes, 0) < n ? 1.0f : 0.0f;
        }
      t.mean /= fmaxf(t.n, 1.0f);
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (column<W, false>(k, e, threadIdx.x, kLongLanes, 0) < n) t.m2 = fmaf(v[k][e] - t.mean, v[k][e] - t.mean, t.m2);
      m = join(m, t);
    }
    m = join_warp(m);
    if (lane == 0) sh[threadIdx.x >> 5] = m;
    __syncthreads();
    m = join_warp(sh[lane]);
    if (threadIdx.x == 0) mine = m;
    cluster.sync();
    m = join_warp(lane < blocks ? *cluster.map_shared_rank(&mine, lane) : Moments{0.0f, 0.0f, 0.0f});
    const float rstd = 1.0f / sqrtf(m.m2 / (float)cols + eps);
    for (int64_t r = rank; r < runs; r += blocks) {
      const int n = cols - r * kLongRun < kLongRun ? (int)(cols - r * kLongRun) : (int)kLongRun;
      load_row<W, NV>(px + r * kLongRun * xr.sc, xr.sc, n, threadIdx.x, kLongLanes, 0.0f, v);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        float wv[W], bv[W];
        load_weight<W, false>(w, wtype, r * kLongRun, 0, n, k, threadIdx.x, kLongLanes, 0, 1.0f, wv);
        load_weight<W, false>(b, wtype, r * kLongRun, 0, n, k, threadIdx.x, kLongLanes, 0, 0.0f, bv);
#pragma unroll
        for (int e = 0; e < W; ++e) v[k][e] = fmaf((v[k][e] - m.mean) * rstd, wv[e], bv[e]);
      }
      store_row<W, NV>(py + r * kLongRun * yr.sc, yr.sc, n, threadIdx.x, kLongLanes, v);
    }
    if (threadIdx.x == 0 && rank == 0) {
      if (mean_out) mean_out[i] = m.mean;
      if (rstd_out) rstd_out[i] = rstd;
    }
    cluster.sync();  // the others have read `mine`, and sh may be written again
  }
}

// ---- launches ---------------------------------------------------------------------
template <class TX, class TY, int NV, int R, int MAXT, bool WRAPS, bool APART>
cudaError_t stream_rows_as(const LayerNormProblem &p, int lanes, int most, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, bytes = kStages<MAXT> * R * Source<W, NV, MAXT, APART, TX>::kBytes;
  auto kernel = ln_forward_stream<TX, TY, W, NV, R, MAXT, WRAPS, APART>;
  if (cudaError_t e = allow_shared(kernel, bytes)) return e;
  const int groups = MAXT / lanes, grid = stream_grid(p.rows, groups, most, W);
  const int64_t step = (int64_t)grid * groups;
  kernel<<<grid, MAXT, bytes, s>>>(static_cast<const TX *>(p.x), row_walk(p.xr, step), static_cast<TY *>(p.y),
                                   row_walk(p.yr, step), p.w, p.b, p.wtype, p.rows, (int)p.cols, p.eps, p.mean, p.rstd, lanes);
  return cudaGetLastError();
}

template <class TX, class TY, int NV, int R, int MAXT, bool APART>
cudaError_t stream_rows(const LayerNormProblem &p, int lanes, int most, cudaStream_t s) {
  if (APART || p.rows > p.xr.n1 || p.rows > p.yr.n1) return stream_rows_as<TX, TY, NV, R, MAXT, true, APART>(p, lanes, most, s);
  return stream_rows_as<TX, TY, NV, R, MAXT, APART, APART>(p, lanes, most, s);
}

// Streamed rows: as many blocks as are resident, or one for each block of rows
// where those are fewer (then one row at a time).
template <class TX, class TY, bool APART>
cudaError_t forward_streamed(const LayerNormProblem &p, int spare, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, NV = kMost / W;
  if (p.cols + spare > kHeld) {
    if (p.rows <= device_sms()) return stream_rows<TX, TY, NV, 1, kHalfLanes, APART>(p, kHalfLanes, device_sms(), s);
    return stream_rows<TX, TY, NV, 2, kHalfLanes, APART>(p, kHalfLanes, device_sms(), s);
  }
  int lanes = row_lanes(p.rows, p.cols, W, kMost, spare);
  if (APART && lanes < 8) lanes = 8;
  const int groups = kThreads / lanes;
  const int nv = row_vectors(p.cols + spare, lanes, W), most = (nv * W > 8 ? 2 : 3) * device_sms();
  if (nv == 1) return stream_rows<TX, TY, 1, 1, kThreads, APART>(p, lanes, most, s);
  if (nv < NV) return stream_rows<TX, TY, 2, 1, kThreads, APART>(p, lanes, most, s);
  if constexpr (sizeof(TX) == 2)
    if (p.rows > (int64_t)most * groups) return stream_rows<TX, TY, NV, 2, kThreads, APART>(p, lanes, most, s);
  return stream_rows<TX, TY, NV, 1, kThreads, APART>(p, lanes, most, s);
}

template <class TX, class TY, bool WRAPS, bool APART>
cudaError_t forward_spread(const LayerNormProblem &p, int blocks, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, bytes = kSpreadStages<TX, APART> * kSpreadRows<TX> * Source<W, kMost / W, kThreads, APART, TX>::kBytes;
  auto kernel = ln_forward_spread<TX, TY, W, WRAPS, APART>;
  if (cudaError_t e = allow_shared(kernel, bytes)) return e;
  int most = 0;
  if (cudaError_t e = resident_clusters(kernel, blocks, kThreads, bytes, &most)) return e;
  const int clusters = stream_grid(p.rows, 1, most, APART ? W : row_period(p.xr, p.rows, W));
  return launch_clusters(kernel, clusters, blocks, kThreads, bytes, s, static_cast<const TX *>(p.x), row_walk(p.xr, clusters),
                         static_cast<TY *>(p.y), row_walk(p.yr, clusters), p.w, p.b, p.wtype, p.rows, (int)p.cols, p.eps, p.mean,
                         p.rstd, blocks);
}

template <class TX, class TY, bool WRAPS, bool APART>
cudaError_t forward_cut(const LayerNormProblem &p, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, bytes1 = kCutStages * kRun * (int)sizeof(TX);
  constexpr int bytes2 = kCutStages * Source<W, kCutMost / W, kThreads, APART, TX>::kBytes;
  auto first = ln_moments<TX, W, WRAPS>;
  auto second = ln_outputs<TX, TY, W, WRAPS, APART>;
  if (cudaError_t e = allow_shared(first, bytes1)) return e;
  if (cudaError_t e = allow_shared(second, bytes2)) return e;
  const int64_t runs = most_runs(p.cols), batch = batch_rows(p.rows, p.cols, sizeof(TX));
  const int period_x = row_period(p.xr, p.rows, W), period = APART && row_period(p.yr, p.rows, W) > 1 ? W : period_x;
  const int parts1 = cut_parts(batch, runs, 4 * device_sms(), period_x), parts2 = cut_parts(batch, runs, 2 * device_sms(), period);
  float4 *shares = static_cast<float4 *>(p.ws);
  for (int64_t row = 0; row < p.rows; row += batch) {
    const int64_t last = row + batch < p.rows ? row + batch : p.rows;
    if (cudaError_t e = launch(row == 0, first, grid_for(runs * parts1), kThreads, bytes1, s, static_cast<const TX *>(p.x),
                               row_walk(p.xr, parts1), p.cols, Cut{row, last, runs, parts1}, shares))
      return e;
    if (cudaError_t e = launch(false, second, grid_for(runs * parts2), kThreads, bytes2, s, static_cast<const TX *>(p.x),
                               row_walk(p.xr, parts2), static_cast<TY *>(p.y), row_walk(p.yr, parts2), p.w, p.b, p.wtype,
                               p.cols, p.eps, p.mean, p.rstd, Cut{row, last, runs, parts2}, shares))
      return e;
  }
  return cudaSuccess;
}

template <class TX, class TY, int NV>
cudaError_t strided_rows(const LayerNormProblem &p, int lanes, cudaStream_t s) {
  const int64_t groups = kThreads / lanes;
  ln_forward<TX, TY, kWidth<TX, TY>, NV><<<grid_for((p.rows + groups - 1) / groups), kThreads, 0, s>>>(
      static_cast<const TX *>(p.x), p.xr, static_cast<TY *>(p.y), p.yr, p.w, p.b, p.wtype, p.rows, (int)p.cols, p.eps, p.mean,
      p.rstd, lanes);
  return cudaGetLastError();
}

template <class TX, class TY>
cudaError_t long_rows(const LayerNormProblem &p, cudaStream_t s) {
  int cluster = 1;
  while (cluster < kCluster && p.cols > kLongRun * cluster) cluster *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((p.rows < (1 << 24) ? p.rows : (1 << 24)) * cluster));
  cfg.blockDim = dim3(kLongLanes);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, ln_forward_long<TX, TY, kWidth<TX, TY>>, static_cast<const TX *>(p.x), p.xr,
                            static_cast<TY *>(p.y), p.yr, p.w, p.b, p.wtype, p.rows, p.cols, p.eps, p.mean, p.rstd);
}

template <class TX, class TY>
cudaError_t forward(const LayerNormProblem &p, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, NV = kMost / W;
  if (steady(p.xr, p.rows, W) && steady(p.yr, p.rows, W)) {
    const int spare = vec_rows(p.y, p.yr, p.rows, sizeof(TY), W) ? 0 : W - 1;
    const bool held = p.cols + spare <= kHalfHeld;
    if (!held && p.cols + spare <= kSpread * kHeld) {
      const int blocks = spread_blocks(p.cols + spare);
      if (!same_shift(p.x, p.xr, sizeof(TX), p.y, p.yr, sizeof(TY), p.rows, W)) return forward_spread<TX, TY, true, true>(p, blocks, s);
      return p.rows > p.xr.n1 || p.rows > p.yr.n1 ? forward_spread<TX, TY, true, false>(p, blocks, s)
                                                  : forward_spread<TX, TY, false, false>(p, blocks, s);
    }
    if (!same_shift(p.x, p.xr, sizeof(TX), p.y, p.yr, sizeof(TY), p.rows, W))
      return held ? forward_streamed<TX, TY, true>(p, spare, s) : forward_cut<TX, TY, true, true>(p, s);
    return held ? forward_streamed<TX, TY, false>(p, spare, s)
           : p.rows > p.xr.n1 || p.rows > p.yr.n1 ? forward_cut<TX, TY, true, false>(p, s)
                                                  : forward_cut<TX, TY, false, false>(p, s);
  }
  if (p.cols > kHeld) return long_rows<TX, TY>(p, s);
  const int lanes = row_lanes(p.rows, p.cols, W, kMost, 0), nv = row_vectors(p.cols, lanes, W);
  if (nv == 1) return strided_rows<TX, TY, 1>(p, lanes, s);
  if (nv < NV) return strided_rows<TX, TY, 2>(p, lanes, s);
  return strided_rows<TX, TY, NV>(p, lanes, s);
}

}  // namespace

size_t layer_norm_forward_workspace_bytes(int64_t rows, int64_t cols) {
  if (cols <= kSpread * kHeld - 7) return 0;
  return (size_t)batch_rows(rows, cols, 2) * (size_t)most_runs(cols) * sizeof(float4);
}

cudaError_t launch_layer_norm(const LayerNormProblem &p, cudaStream_t s) {
  return by_types(p.xtype, p.ytype, [&](auto tx, auto ty) { return forward<decltype(tx), decltype(ty)>(p, s); });
}

}  // namespace spmdb200
