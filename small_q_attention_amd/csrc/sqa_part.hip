// gfx950 kernels of attention over a part of every sequence's pages, and the join of the
// partial rows that a sequence's splits leave.
//
// Row i of sequence b stands at p = seq_lens[b] - Q + i. With a window W and S first tokens
// it sees token t if the draft rule lets it and (t < S or t > p - W):
//   out(row) = sum_t 2^(c s(row, t)) v_t / sum_t 2^(c s(row, t)),  c = scale log2(e)
// Under a shared prefix a sequence's own splits are what follows the shared pages. Either
// way a sequence is a list of pages, [0, head) and [tail, ..), of which the first and the
// last few are masked, cut into splits; with (m, l, O) the maximum, sum and unnormalised
// output of a split's tokens, splits join as
//   m = max_j m_j,  l = sum_j l_j 2^(m_j - m),  O = sum_j O_j 2^(m_j - m).
#include "sqa_part.h"
#include "sqa_part_device.h"

namespace sqa {
namespace {

// Joins the partial rows of every output row: a sequence's own splits and, where it shares
// a prefix, its group's. One wave per row, (HD / 4) lanes across a partial row and the
// row's splits dealt over the lane groups; weights in lane j for split j. Rows that one
// split has left in the output are skipped.
template <int HD, typename E>
__global__ __launch_bounds__(256) void sqa_join_kernel(PartArgs args) {
  const PartialArgs& a = args.p;
  constexpr int CH = HD / 4 < 64 ? HD / 4 : 64;  // lanes across a row
  constexpr int SG = 64 / CH;                    // splits at a time
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * 4 + wave;
  if (row >= a.batch * a.q_len * a.hq) return;
  const int token = row / a.hq, h = row - token * a.hq;
  const int b = token / a.q_len, qi = token - b * a.q_len;
  const int kvh = h / a.by_group;
  const int r = qi * a.group + h - kvh * a.group;
  const int len = max(scalar_load(a.seq_lens + b), 0);
  const Span span = span_of(args, b, len);
  int own, first;
  if (args.splits > 0) {
    int size;
    own_splits(args, span.n, &own, &size);
    first = b * args.splits;
    if (span.before < 0 && own <= 1) return;  // uniform: in the output
  } else {
    const SeqSplits t = a.seq_splits[b];
    own = t.count;
    first = t.first;
    if (span.before < 0 && own == 1) return;  // uniform: in the output
  }
  own = __builtin_amdgcn_readfirstlane(own);
  int shared = 0, slot = 0;
  if (span.before >= 0) {  // uniform
    int size;
    even_splits(span.shared, args.shared_size, &shared, &size);
    slot = shared_slot(args, b, span.before);
    shared = __builtin_amdgcn_readfirstlane(
        min(shared, args.packed ? args.shared_slots - slot : args.most_splits));
  }
  const int total = own + shared;
  const long long own_at = ((long long)first * a.hkv + kvh) * a.rows + r;
  const long long group_at = args.shared_at + ((long long)slot * a.hkv + kvh) * a.rows + r;
  const long long step = (long long)a.hkv * a.rows;
  auto place = [&](int j) {
    return j < own ? own_at + j * step : group_at + (j - own) * step * args.slot_step;
  };
  const int c = lane % CH, sg = lane / CH;
  float m = -INFINITY, l = 0.f;
  f4 acc = {0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;
  for (int j0 = 0; j0 < total; j0 += 64) {
    const int n = min(total - j0, 64);
    auto fetch = [&](int k, f4 (&o)[U]) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        o[u] = *(const f4*)(a.part_o + place(j0 + min(k + u * SG + sg, n - 1)) * HD + 4 * c);
    };
    const int j = min(j0 + lane, total - 1);
    const float2 ml = *(const float2*)(a.part_ml + place(j) * 2);
    f4 o[U];
    fetch(0, o);  // on their way beside the maxima
    const bool is = j0 + lane < total;
    float top = is && ml.y != 0.f ? ml.x : -INFINITY;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
    const float mn = fmaxf(m, top);
    const float base = mn == -INFINITY ? 0.f : mn;
    // A NaN sum counts whatever the maxima; of a split that saw no key the sums are 0.
    const float w = is ? (ml.y != ml.y ? 1.f : weight_of(ml.x - base)) : 0.f;
    float ls = is ? w * ml.y : 0.f;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) ls += __shfl_xor(ls, o);
    const float alpha = weight_of(m - base);
    l = l * alpha + ls;
    acc *= alpha;
    m = mn;
    for (int k = 0; k < n; k += U * SG) {
      if (k > 0) fetch(k, o);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = k + u * SG + sg;
        const float x = __shfl(w, min(at, 63));
        if (at < n) acc += o[u] * x;
      }
    }
  }
  if constexpr (SG > 1) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int o = CH; o < 64; o *= 2) acc[e] += __shfl_xor(acc[e], o);
  }
  const float inv = l != 0.f ? a.out_scale / l : 0.f;
  if (sg == 0) {
    const float o[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
    *(u2*)(a.out + (long long)row * HD + 4 * c) = E::pack4(o);
  }
}

}  // namespace

hipError_t launch_own(const PartArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)own_workgroups(a));
  if (a.p.bf16)
    launch_part<ElemBF16, false>(a, a.p.rows, grid, stream);
  else
    launch_part<ElemF16, false>(a, a.p.rows, grid, stream);
  return hipGetLastError();
}

template <typename E>
void launch_join_as(const PartArgs& a, dim3 grid, hipStream_t stream) {
  if (a.p.head_dim == 64)
    hipLaunchKernelGGL((sqa_join_kernel<64, E>), grid, dim3(256), 0, stream, a);
  else if (a.p.head_dim == 128)
    hipLaunchKernelGGL((sqa_join_kernel<128, E>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((sqa_join_kernel<256, E>), grid, dim3(256), 0, stream, a);
}

hipError_t launch_join(const PartArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)(((long long)a.p.batch * a.p.q_len * a.p.hq + 3) / 4));
  if (a.p.bf16)
    launch_join_as<ElemBF16>(a, grid, stream);
  else
    launch_join_as<ElemF16>(a, grid, stream);
  return hipGetLastError();
}

}  // namespace sqa
