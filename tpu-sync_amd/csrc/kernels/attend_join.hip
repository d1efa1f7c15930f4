// Joins the parts of attention rows whose keys were split, or read with a
// group's: with (m, l, o) of each part, o relative to its maximum m,
//   M = max m,  out = sum o e^{m - M} / sum l e^{m - M},  lse = M + log sum l e^{m - M}.
// A workgroup takes a row at a time, a part to every head_dim / 4 threads, so
// a row of many parts (one long sequence) is read at once; parts are merged in
// a fixed order. Rows that attend_few or attend_many finished are not visited.
#include "attend_plan.h"

namespace kvx {
namespace {

struct Merged {
  float m = -__builtin_inff(), l = 0.0f;
  f32x4 v = {0, 0, 0, 0};

  __device__ __forceinline__ void Add(float pm, float pl, f32x4 pv) {
    const float now = fmaxf(m, pm);
    const float back = now == -__builtin_inff() ? 0.0f : now;
    const float f = __builtin_amdgcn_exp2f(m - back), g = __builtin_amdgcn_exp2f(pm - back);
    m = now;
    l = l * f + pl * g;
    v = v * f + pv * g;
  }
};

template <class E>
__global__ __launch_bounds__(kAttendThreads) void attend_join_kernel(const AttendLaunch a) {
  extern __shared__ __align__(16) char lds[];
  __shared__ f32x4 part_v[kAttendThreads];
  __shared__ f32x2 part_s[kAttendThreads];
  using Scalar = typename E::Scalar;
  const BatchView& b = a.batch;
  const int S = b.sequences, units = a.groups + S, G = a.q_heads / a.k_heads;
  int* few = reinterpret_cast<int*>(lds);  // [sequences] steps of attend_few
  int* many = few + S;                     // [groups + sequences] items of attend_many
  int* todo = many + units;                // [sequences] rows to join
  const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  const auto unit_of = [&](int i) {
    return i < a.groups ? LoadGroup(a, i) : LoadManySequence(LoadOwnKeys(a, i - a.groups));
  };
  int few_all = 0;
  if (a.few_grid > 0) {
    for (int s = threadIdx.x; s < S; s += kAttendThreads) few[s] = FewSteps(LoadOwnKeys(a, s));
    BlockSums(few, S);
    few_all = one(few[S - 1]);
  }
  int each = 0;
  if (a.many_grid > 0) {
    for (int i = threadIdx.x; i < units; i += kAttendThreads) many[i] = ManyTiles(unit_of(i));
    BlockSums(many, units);
    const int tiles = one(many[units - 1]) * a.k_heads;
    if (tiles > 0 && tiles < a.many_target) {
      __syncthreads();
      for (int i = threadIdx.x; i < units; i += kAttendThreads) {
        const ManyUnit u = unit_of(i);
        many[i] = ManyTiles(u) * ManySteps(u);
      }
      BlockSums(many, units);
      each = ManyEach(a, tiles, static_cast<int64_t>(one(many[units - 1])) * a.k_heads);
      __syncthreads();
      for (int i = threadIdx.x; i < units; i += kAttendThreads) {
        const ManyUnit u = unit_of(i);
        many[i] = ManyTiles(u) * ManyParts(ManySteps(u), each);
      }
      BlockSums(many, units);
    }
  }
  const FewAxis axis(a, max(few_all, 1));
  for (int s = threadIdx.x; s < S; s += kAttendThreads) {
    const OwnKeys k = LoadOwnKeys(a, s);
    bool split = k.grouped;
    if (k.rows > 0 && k.rows <= kFewRows && few_all > 0) {
      const int x0 = (s > 0 ? few[s - 1] : 0) * a.k_heads, x1 = few[s] * a.k_heads;
      split = split || axis.Owner(x0) != axis.Owner(x1 - 1);
    } else if (k.rows > kFewRows) {
      split = split || ManyParts(ManySteps(LoadManySequence(k)), each) > 1;
    }
    todo[s] = split ? k.rows * a.k_heads : 0;
  }
  BlockSums(todo, S);
  const int all = one(todo[S - 1]);

  const int lanes = a.padded_dim / 4;
  const int at_once = kAttendThreads / lanes;  // parts
  const int mine = threadIdx.x / lanes, d = threadIdx.x % lanes * 4;
  for (int j = blockIdx.x; j < all; j += gridDim.x) {
    const int s = one(FirstAbove(todo, S, j));
    const OwnKeys k = LoadOwnKeys(a, s);
    const int rest = j - (s > 0 ? one(todo[s - 1]) : 0);
    const int rows = one(k.rows);
    const int h = rest / rows, row = rest - h * rows;
    const int t = FastDivI(a.group_div, row);
    const int64_t token = k.q.first + t;
    const int head = h * G + (row - t * G);

    // The row's parts: `own` of them, then `shared` of its group's prefix.
    int own = 0, shared = 0, w0 = 0, x0 = 0;
    int64_t own_row = 0, own_step = 0, shared_row = 0, shared_step = 0;
    const bool is_few = rows <= kFewRows;
    if (is_few) {
      const int steps = one(few[s] - (s > 0 ? few[s - 1] : 0));
      x0 = (s > 0 ? one(few[s - 1]) : 0) * a.k_heads + h * steps;
      w0 = axis.Owner(x0);
      own = axis.Owner(x0 + steps - 1) - w0 + 1;
      own_row = row;
    } else {
      const ManyUnit u = LoadManySequence(k);
      const int tiles = ManyTiles(u), i = a.groups + s;
      own = ManyParts(ManySteps(u), each);
      own_row = ManySlotRow(a, (i > 0 ? many[i - 1] : 0) * a.k_heads +
                                   h * own * tiles + (tiles - 1 - row / kManyRows)) +
                row % kManyRows;
      own_step = static_cast<int64_t>(tiles) * kManyRows;
    }
    if (k.grouped) {
      const int g = GroupOf(a, s);
      const ManyUnit u = LoadGroup(a, g);
      if (u.rows > 0) {
        const int tiles = ManyTiles(u), r = (static_cast<int>(token) - u.first) * G + (row - t * G);
        shared = ManyParts(ManySteps(u), each);
        shared_row = ManySlotRow(a, (g > 0 ? many[g - 1] : 0) * a.k_heads + h * shared * tiles +
                                        (tiles - 1 - r / kManyRows)) +
                     r % kManyRows;
        shared_step = static_cast<int64_t>(tiles) * kManyRows;
      }
    } else if (own == 1) {
      continue;  // this key head's keys were not cut
    }
    Merged sum;
    if (mine < at_once) {
#pragma unroll 4
      for (int n = mine; n < own + shared; n += at_once) {
        int64_t from;
        if (n >= own) {
          from = shared_row + (n - own) * shared_step;
        } else if (is_few && own == 1) {
          from = WholeRow(a, token, head);
        } else if (is_few) {
          const int w = w0 + n;
          from = FewSlotRow(a, n == 0 && axis.Start(w) != x0 ? 2 * w + 1 : 2 * w) + own_row;
        } else {
          from = own_row + n * own_step;
        }
        const f32x2 st = PartStats(a)[from];
        sum.Add(st[0], st[1], *reinterpret_cast<const f32x4*>(a.parts + from * a.padded_dim + d));
      }
      part_v[threadIdx.x] = sum.v;
      part_s[threadIdx.x] = f32x2{sum.m, sum.l};
    }
    __syncthreads();
    if (mine == 0) {
      for (int n = 1; n < min(at_once, own + shared); ++n) {
        const f32x2 st = part_s[n * lanes + threadIdx.x];
        sum.Add(st[0], st[1], part_v[n * lanes + threadIdx.x]);
      }
      if (d < a.head_dim) {
        const float inverse = sum.l > 0.0f ? 1.0f / sum.l : (sum.l == 0.0f ? 0.0f : sum.l);
        using Pair = u32x2 __attribute__((aligned(2)));
        *reinterpret_cast<Pair*>(static_cast<Scalar*>(a.out) + token * a.out_token +
                                 head * a.out_head + d) =
            u32x2{Pack2<E>(sum.v[0] * inverse, sum.v[1] * inverse),
                  Pack2<E>(sum.v[2] * inverse, sum.v[3] * inverse)};
      }
      if (a.lse != nullptr && d == 0) {
        a.lse[token * a.q_heads + head] = (sum.m + log2f(sum.l)) / kLog2e;
      }
    }
    __syncthreads();
  }
}

int64_t CeilDiv(int64_t n, int64_t d) { return (n + d - 1) / d; }

}  // namespace

hipError_t LaunchAttendJoin(const AttendLaunch& l, hipStream_t stream) {
  const int64_t rows = static_cast<int64_t>(l.batch.tokens) * l.q_heads;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(rows, 2048));
  const size_t lds = static_cast<size_t>(3 * l.batch.sequences + l.groups) * sizeof(int);
  if (l.type == kBf16) {
    hipLaunchKernelGGL(attend_join_kernel<Bf16>, dim3(grid), dim3(kAttendThreads), lds, stream, l);
  } else {
    hipLaunchKernelGGL(attend_join_kernel<F16>, dim3(grid), dim3(kAttendThreads), lds, stream, l);
  }
  return hipGetLastError();
}

int64_t PlanAttend(AttendLaunch* l) {
  constexpr int kCus = 256;
  const int64_t G = l->q_heads / l->k_heads;
  const int64_t T = l->batch.tokens, S = l->batch.sequences;
  const bool single = l->batch.starts == nullptr;
  l->padded_dim = l->head_dim <= 64 ? 64 : l->head_dim <= 96 ? 96 : l->head_dim <= 128 ? 128 : 256;
  l->few_grid = l->many_grid = l->many_parts = 0;
  l->part_rows = 0;
  // Rows of one sequence that may meet attend_few.
  const int64_t most = single ? G : std::min<int64_t>(T * G, kFewRows);
  const bool full = l->head_dim == l->padded_dim;
  l->few_rows = most <= 16 && full ? 16 : 32;
  if (G <= kFewRows) {
    const int per_cu = l->padded_dim > 128 ? 1 : l->few_rows == 16 ? 3 : 2;
    const int64_t steps = S * l->k_heads * CeilDiv(std::max(l->batch.capacity, 1), kFewStep);
    l->few_grid = static_cast<int>(std::min<int64_t>(kCus * per_cu, steps));
  }
  const bool many_sequences = single ? G > kFewRows : T * G > kFewRows;
  if (many_sequences || l->groups > 0) {
    l->many_target = l->padded_dim > 128 ? kCus : 2 * kCus;
    int64_t tiles = 0;
    if (many_sequences) tiles += CeilDiv(T * G, kManyRows) + std::min(S, T * G / (kFewRows + 1));
    if (l->groups > 0) tiles += CeilDiv(T * G, kManyRows) + l->groups;
    tiles *= l->k_heads;
    const int64_t split = std::min<int64_t>(2 * l->many_target, l->many_target + tiles);
    const int64_t steps = CeilDiv(std::max(l->batch.capacity, 1), kManyStep);
    l->many_grid = static_cast<int>(std::min(std::max(tiles, split), tiles * CeilDiv(steps, 8)));
    l->many_parts = l->groups > 0 ? l->many_grid
                                  : static_cast<int>(std::min<int64_t>(l->many_grid, split));
  }
  l->join = l->groups > 0 || l->batch.capacity > kFewStep;
  if (!l->join) return 0;
  l->part_rows = 2ll * l->few_grid * l->few_rows +
                 static_cast<int64_t>(l->many_parts) * kManyRows +
                 (l->groups > 0 ? T * l->q_heads : 0);
  return l->part_rows * (l->padded_dim + 2) * static_cast<int64_t>(sizeof(float));
}

hipError_t LaunchAttend(const AttendLaunch& l, hipStream_t stream) {
  hipError_t e = hipSuccess;
  if (l.many_grid > 0) e = LaunchAttendMany(l, stream);
  if (e == hipSuccess && l.few_grid > 0) e = LaunchAttendFew(l, stream);
  if (e == hipSuccess && l.join) e = LaunchAttendJoin(l, stream);
  return e;
}

}  // namespace kvx
