// Joins the parts of attention rows whose keys were split, or read with a
// group's: with (m, l, o) of each part, o relative to its maximum m,
//   M = max m,  out = sum o e^{m - M} / sum l e^{m - M},  lse = M + log sum l e^{m - M}.
// The cuts are found from the plan that the kernel before this one left: a row's
// keys were cut where a worker's part starts inside them. A workgroup takes
// join_rows rows of one sequence and key head at a time, a part to every head_dim
// / 4 threads, so a row of many parts (one long sequence) is read at once; parts
// are merged in a fixed order. Rows that were finished are not visited. Reading
// the parts bounds it where there are many (67 MB written and read for 4099 new
// tokens of 32 heads: 37 us), its launch and the plan's loads where there are few
// (one sequence of 700 tokens: 6 us).
#include <algorithm>

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
  int* words = reinterpret_cast<int*>(lds);
  const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  const int* from = Plan(a);
  for (int i = threadIdx.x; i < PlanWords(a); i += kAttendThreads) words[i] = from[i];
  __syncthreads();
  const PlanView plan(a, words);
  const Axis few = FewAxis(a, one(plan.few[S - 1]));
  const Axis many = ManyAxis(a, one(plan.many[units - 1]));
  const auto before = [](const int* sums, int i) { return i > 0 ? sums[i - 1] : 0; };

  const int lanes = a.padded_dim / 4, d = threadIdx.x % lanes * 4;
  const int team = threadIdx.x / lanes;  // threads of one part's row
  const int at_once = kAttendThreads / lanes / a.join_rows;  // parts
  const int mine = team / a.join_rows, in_group = team % a.join_rows;

  // Items: the row groups of what may have been cut. Few rows: every (sequence,
  // key head), or what each worker's start is in, where that is less; then many
  // rows: the tile that each worker's start is in, behind the groups' prefixes;
  // then the grouped sequences, whose rows all have a part of the prefix.
  const int few_shift = 32 - __clz(max((a.few_rows - 1) / a.join_rows, 0));
  const int many_shift = 31 - __clz(kManyRows / a.join_rows);
  const bool by_cut = few.workers <= S * a.k_heads;
  const int few_items = (by_cut ? max(few.workers - 1, 0) : few.total > 0 ? S * a.k_heads : 0)
                        << few_shift;
  const int many_first = a.groups > 0 ? many.Owner(before(plan.many, a.groups) * a.k_heads) : 0;
  const int many_items = max(many.workers - 1 - many_first, 0) << many_shift;
  const int items = few_items + many_items + one(plan.todo[S - 1]) * a.k_heads;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    int s, h, row0;           // sequence, key head, first row
    int x = 0, size = 0;      // the rows' place on their axis
    const bool is_cut = item < few_items + many_items;
    bool is_few = item < few_items;
    if (is_few) {
      const int n = item >> few_shift, cut = few.Start(n + 1);
      s = by_cut ? one(FirstAbove(plan.few, S, cut / a.k_heads)) : n / a.k_heads;
      const int at = one(before(plan.few, s));
      size = one(plan.few[s]) - at;
      if (size == 0) continue;
      h = by_cut ? (cut - at * a.k_heads) / size : n - s * a.k_heads;
      x = at * a.k_heads + h * size;
      row0 = (item & ((1 << few_shift) - 1)) * a.join_rows;
      // The first cut inside takes it.
      if (by_cut && (cut == x || cut - few.each > x)) continue;
    } else if (is_cut) {
      const int n = item - few_items, cut = many.Start(many_first + (n >> many_shift) + 1);
      const int i = one(FirstAbove(plan.many, units, cut / a.k_heads));
      if (i < a.groups) continue;  // with its sequences, below
      s = i - a.groups;
      const int at = one(before(plan.many, i)), per_head = one(plan.many[i]) - at;
      const int base = one(plan.base[i]), tiles = (one(plan.rows[s]) + kManyRows - 1) / kManyRows;
      h = (cut - at * a.k_heads) / per_head;
      const int unit = at * a.k_heads + h * per_head;
      const int tile = one(TileAt(a, false, base, tiles, cut - unit));
      x = unit + ManyCost(a, false, base, tile);
      size = unit + ManyCost(a, false, base, tile + 1) - x;
      row0 = tile * kManyRows + (n & ((1 << many_shift) - 1)) * a.join_rows;
      if (cut == x || cut - many.each > x) continue;
    } else {
      const int n = item - few_items - many_items;
      s = one(FirstAbove(plan.todo, S, n / a.k_heads));
      const int rest = n - one(before(plan.todo, s)) * a.k_heads;
      h = rest % a.k_heads;
      row0 = rest / a.k_heads * a.join_rows;
      is_few = one(plan.rows[s]) <= kFewRows;
      if (is_few) {
        const int at = one(before(plan.few, s));
        size = one(plan.few[s]) - at;
        x = at * a.k_heads + h * size;
      } else {
        const int i = a.groups + s, at = one(before(plan.many, i)), base = one(plan.base[i]);
        const int tile = row0 / kManyRows;
        x = at * a.k_heads + h * (one(plan.many[i]) - at) + ManyCost(a, false, base, tile);
        size = ManyCost(a, false, base, tile + 1) - ManyCost(a, false, base, tile);
      }
    }
    const int rows = one(plan.rows[s]), g = one(plan.group[s]);
    if (row0 >= rows || (is_cut && g >= 0)) continue;
    const int row = min(row0 + in_group, rows - 1);
    const bool has_row = row0 + in_group < rows;
    const int t = FastDivI(a.group_div, row);
    const int64_t token = one(plan.first[s]) + t;
    const int head = h * G + (row - t * G);

    // The row's parts: workers [w0, w0 + own) of its own keys' axis and, of a
    // group's, [v0, v0 + shared) of the prefix's. (Starts or groups that are out
    // of order may point behind the axes: bounded, their rows mean nothing.)
    const Axis& axis = is_few ? few : many;
    const int w0 = axis.Owner(x), own = axis.Owner(x + size - 1) - w0 + 1;
    if (g < 0 && own == 1) continue;
    int shared_row = 0, y = 0, v0 = 0, shared = 0;
    if (g >= 0) {
      const int at = before(plan.many, g), per_head = plan.many[g] - at;
      if (per_head > 0) {
        shared_row = max((static_cast<int>(token) - plan.gfirst[g]) * G + (row - t * G), 0);
        const int tile = shared_row / kManyRows, base = plan.base[g];
        y = at * a.k_heads + h * per_head + ManyCost(a, true, base, tile);
        v0 = many.Owner(y);
        shared = many.Owner(y + base - 1) - v0 + 1;
      }
    }
    Merged sum;
    if (mine < at_once) {
#pragma unroll 4
      for (int n = mine; n < own + shared; n += at_once) {
        int64_t from;
        if (n >= own) {
          const int w = max(min(v0 + n - own, many.workers - 1), 0);
          from = shared == 1 ? WholeRow(a, true, token, head)
                             : ManySlotRow(a, n == own ? many.Slot(w, y) : 2 * w) +
                                   shared_row % kManyRows;
        } else if (own == 1) {
          from = WholeRow(a, false, token, head);
        } else {
          const int w = max(min(w0 + n, axis.workers - 1), 0);
          const int slot = n == 0 ? axis.Slot(w, x) : 2 * w;
          from = is_few ? FewSlotRow(a, slot) + row : ManySlotRow(a, slot) + row % kManyRows;
        }
        const f32x2 st = PartStats(a)[from];
        sum.Add(st[0], st[1], *reinterpret_cast<const f32x4*>(a.parts + from * a.padded_dim + d));
      }
      part_v[threadIdx.x] = sum.v;
      part_s[threadIdx.x] = f32x2{sum.m, sum.l};
    }
    __syncthreads();
    if (mine == 0) {
      for (int n = 1; n < at_once; ++n) {
        const int other = n * a.join_rows * lanes + threadIdx.x;
        const f32x2 st = part_s[other];
        sum.Add(st[0], st[1], part_v[other]);
      }
      if (has_row && d < a.head_dim) {
        const f32x4 v = sum.v * InverseSum(sum.l);
        using Pair = u32x2 __attribute__((aligned(2)));
        *reinterpret_cast<Pair*>(static_cast<Scalar*>(a.out) + token * a.out_token +
                                 head * a.out_head + d) =
            u32x2{Pack2<E>(v[0], v[1]), Pack2<E>(v[2], v[3])};
      }
      if (has_row && a.lse != nullptr && d == 0) {
        a.lse[token * a.q_heads + head] = (sum.m + log2f(sum.l)) / kLog2e;
      }
    }
    __syncthreads();
  }
}

int64_t CeilDiv(int64_t n, int64_t d) { return (n + d - 1) / d; }

}  // namespace

hipError_t LaunchAttendJoin(const AttendLaunch& l, hipStream_t stream) {
  const size_t lds = PlanWords(l) * sizeof(int);
  constexpr auto bf16 = attend_join_kernel<Bf16>, f16 = attend_join_kernel<F16>;
  const hipError_t e = l.type == kBf16 ? AllowDynamicLds<bf16>(lds) : AllowDynamicLds<f16>(lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(l.type == kBf16 ? bf16 : f16, dim3(l.join_grid), dim3(kAttendThreads), lds,
                     stream, l);
  return hipGetLastError();
}

int64_t PlanAttend(AttendLaunch* l) {
  constexpr int kCus = 256;
  const int64_t G = l->q_heads / l->k_heads;
  const int64_t T = l->batch.tokens, S = l->batch.sequences;
  const int64_t capacity = std::max(l->batch.capacity, 1);
  const bool single = l->batch.starts == nullptr;
  l->padded_dim = PaddedDim(l->head_dim);
  l->few_grid = l->few_rows = l->many_grid = l->join_grid = l->join_rows = 0;
  l->part_rows = 0;
  const int resident = (l->padded_dim > 128 ? 1 : 2) * kCus;  // workgroups
  if (G <= kFewRows) {
    l->few_rows = static_cast<int>(single ? G : std::min<int64_t>(T * G, kFewRows));
    const int64_t steps = S * l->k_heads * CeilDiv(capacity, kFewStep);
    // One place is left to the plan's workgroup.
    l->few_grid = static_cast<int>(std::min<int64_t>(resident - 1, CeilDiv(steps, kWaves)));
  }
  const bool many_sequences = single ? G > kFewRows : T * G > kFewRows;
  if (many_sequences || l->groups > 0) {
    const int64_t tiles = CeilDiv(T * G, kManyRows) * 2 + S + l->groups;
    const int64_t steps = tiles * l->k_heads * (CeilDiv(capacity, kManyStep) + 2);
    l->many_grid = static_cast<int>(std::min<int64_t>(resident, std::max<int64_t>(steps / kLeastPart, 1)));
  }
  if (l->groups == 0 && l->many_grid == 0 && capacity <= kFewStep) return 0;  // nothing to split
  // Rows that a workgroup joins at once: as many as it has teams of a row's
  // threads, but fewer where that leaves CUs without work.
  const int64_t rows = T * l->q_heads;
  const int teams = l->padded_dim == 64 ? 16 : l->padded_dim <= 128 ? 8 : 4;
  const int64_t most = l->many_grid > 0 ? kManyRows : l->few_rows;
  l->join_rows = 1;
  while (l->join_rows < teams && l->join_rows < most && rows / l->join_rows >= 4 * kCus) {
    l->join_rows *= 2;
  }
  const int64_t units = std::min<int64_t>(S * l->k_heads, kWaves * l->few_grid);
  const int64_t groups = 2 * units * CeilDiv(l->few_rows, l->join_rows) +
                         l->many_grid * CeilDiv(kManyRows, l->join_rows) +
                         (l->groups > 0 ? CeilDiv(rows, l->join_rows) + S * l->k_heads : 0);
  // Four workgroups a CU, each going through its share of the rows: every one
  // loads the plan. 128 sequences on a prefix of 16000: 105 us with 1024
  // workgroups, 107 with 2048, 108 with 512; 28 new tokens of 2 sequences, 40 heads
  // on 8: 26.8, 28.2 and 31.2 us.
  l->join_grid = static_cast<int>(std::min<int64_t>(groups, 4 * kCus));
  l->part_rows = 2ll * kWaves * l->few_grid * l->few_rows + 2ll * l->many_grid * kManyRows +
                 (l->groups > 0 ? 2 * rows : 0);
  return (l->part_rows * (l->padded_dim + 2) + PlanWords(*l)) * static_cast<int64_t>(sizeof(float));
}

hipError_t LaunchAttend(const AttendLaunch& l, hipStream_t stream) {
  hipError_t e = l.many_grid > 0 ? LaunchAttendMixed(l, stream) : LaunchAttendFew(l, stream);
  if (e == hipSuccess && l.join_grid > 0) e = LaunchAttendJoin(l, stream);
  return e;
}

}  // namespace kvx
