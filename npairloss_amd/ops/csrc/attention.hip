// Entry points of attention with capped scores, distance biases and masks (gfx950).
// The mathematics stands in attention.h, the kernels in attention_kernels.h.

#include <torch/extension.h>
#include <ATen/DeviceGuard.h>
#include <ATen/hip/HIPContext.h>

#include "attention_launch.h"

namespace {

// --- ids of 64 rows ---------------------------------------------------------

__global__ __launch_bounds__(WAVE) void doc_ranges_kernel(const int* __restrict__ ids, int L, int tiles,
                                                          DocRange* __restrict__ out) {
  const int b = blockIdx.x / tiles, t = blockIdx.x % tiles, row = t * kDocTile + threadIdx.x;
  const int id = row < L ? ids[static_cast<int64_t>(b) * L + row] : -1;
  const int lo = wave_min(id >= 0 ? id : INT_MAX), hi = wave_max(id);
  const uint64_t there = __ballot(id >= 0);
  if (threadIdx.x == 0) out[blockIdx.x] = DocRange{lo, hi, there};
}

// Blocks of kBlockRows rows in falling order of how many tiles of the other side their ids
// may meet, for each batch row: with packed documents one block has ten times the work of
// another, and the long ones have to begin first.  Two rows of 4096 tokens, 12 heads of 64
// bf16, images of 37 to 785 tokens: dQ 124 -> 82 us, dK and dV 143 -> 95, forward 88 -> 77,
// for 7 us of this kernel a direction.
constexpr int kBlockRows = 2 * kDocTile, kMostOrdered = 1024;

__global__ __launch_bounds__(kMostOrdered) void block_order_kernel(const DocRange* __restrict__ own, int own_tiles, const DocRange* __restrict__ other,
                                                                   int other_tiles, int blocks, int* __restrict__ order) {
  __shared__ int2 staged[kMostOrdered];
  __shared__ int counts[kMostOrdered];
  const int t = threadIdx.x, b = blockIdx.x;
  own += static_cast<int64_t>(b) * own_tiles;
  other += static_cast<int64_t>(b) * other_tiles;
  int lo = INT_MAX, hi = -1, count = 0;
  for (int x = 2 * t; x < min(2 * t + 2, own_tiles); ++x) {
    lo = min(lo, own[x].lo);
    hi = max(hi, own[x].hi);
  }
  for (int base = 0; base < other_tiles; base += blockDim.x) {
    const int n = min(static_cast<int>(blockDim.x), other_tiles - base);
    __syncthreads();
    if (t < n) staged[t] = make_int2(other[base + t].lo, other[base + t].hi);
    __syncthreads();
#pragma unroll 8
    for (int x = 0; x < n; ++x) count += staged[x].x <= hi && staged[x].y >= lo;
  }
  counts[t] = count;
  __syncthreads();
  if (t >= blocks) return;
  int rank = 0;
#pragma unroll 8
  for (int x = 0; x < blocks; ++x) rank += counts[x] > count || (counts[x] == count && x < t);
  order[static_cast<int64_t>(b) * blocks + rank] = t;
}

// The largest of this lane's value and those of higher lanes.
DEVINL float suffix_max(float v) {
#pragma unroll
  for (int off = 1; off < WAVE; off *= 2) v = fmaxf(v, __shfl_down(v, off, WAVE));
  return v;
}

// grad_scale for each key, of 64 keys a workgroup.  A factor of the call's largest |dO| would
// need no kernel, but a large gradient in one document, or in padding, then takes the bits of
// all others' keys.  A key sees the queries of its id from some query on.  Queries that all 64
// keys see go by maxima of 32; in other tiles of 64 lanes are first queries, for each id a
// maximum over those behind every lane, then keys, which take theirs.  8191 tokens, 16 heads on
// 4, causal: 7 us, by rows and not blocks of 32 it was 40; two rows of 4096 packed with images,
// 12 heads: 12 us.
constexpr int kLiftWaves = 4, kLiftRuns = 8;

__global__ __launch_bounds__(kLiftWaves * WAVE) void key_lifts_kernel(AttnArgs a, const DocRange* ranges, int key_tiles) {
  __shared__ float tops[kLiftWaves][WAVE];
  const int t = threadIdx.x, lane = t % WAVE;
  const int wave = __builtin_amdgcn_readfirstlane(t / WAVE);
  const int64_t bc = blockIdx.x / key_tiles;
  const int b = bc / a.Hk, kv = bc % a.Hk, group = a.H / a.Hk, off = a.Lk - a.Lq;
  const int j = static_cast<int>(blockIdx.x % key_tiles) * WAVE + lane;
  const int doc = j < a.Lk && a.k_doc != nullptr ? a.k_doc[static_cast<int64_t>(b) * a.Lk + j] : 0;
  const bool ok = j < a.Lk && doc >= 0;
  // the first query that sees a key
  const int begin = !ok ? INT_MAX : !a.causal || (a.prefix != nullptr && j < a.prefix[b]) ? 0 : max(0, j - off);
  const int least_begin = wave_min(begin), most_begin = wave_max(ok ? begin : 0);
  const int lo = wave_min(ok ? doc : INT_MAX), hi = wave_max(ok ? doc : -1);
  const int q_tiles = (a.Lq + kDocTile - 1) / kDocTile, first_tile = min(least_begin / kDocTile, q_tiles);
  const DocRange* own = ranges != nullptr ? ranges + static_cast<int64_t>(b) * q_tiles : nullptr;
  const int* d0 = a.q_doc != nullptr ? a.q_doc + static_cast<int64_t>(b) * a.Lq : nullptr;
  const int64_t head = static_cast<int64_t>(b) * a.H + kv * group;
  float whole = 0.f, top = 0.f;  // by lanes as queries, by lanes as keys
  auto rows = [&](int i) {       // query i's largest of the heads that share the key
    float m = 0.f;
    if (i < a.Lq) {
#pragma unroll 4
      for (int g = 0; g < group; ++g) m = fmaxf(m, a.row_top[(head + g) * a.Lq + i]);
    }
    return m;
  };
  auto take = [&](float m, int i0, bool mine) {  // of the lanes' rows those that a key sees
    const float from = __shfl(suffix_max(m), max(begin - i0, 0) % WAVE, WAVE);
    if (mine && begin < i0 + WAVE) top = fmaxf(top, from);
  };
  if (own == nullptr) {
    const int whole_tile = max(first_tile, (most_begin + kDocTile - 1) / kDocTile);
    const int tops32 = (a.Lq + 31) / 32, first = min(2 * whole_tile, tops32);
#pragma unroll 4
    for (int x = t; x < group * (tops32 - first); x += kLiftWaves * WAVE)
      whole = fmaxf(whole, a.block_top[(head + x / (tops32 - first)) * tops32 + first + x % (tops32 - first)]);
    for (int n = first_tile + wave; n < min(whole_tile, q_tiles); n += kLiftWaves) take(rows(n * kDocTile + lane), n * kDocTile, ok);
  } else {
    TileWalk walk(own, lo, hi, first_tile, q_tiles);
    int turn = 0;
    for (int n = walk.next(); n >= 0; n = walk.next()) {
      if (turn++ % kLiftWaves != wave) continue;
      const int i0 = n * kDocTile, i = i0 + lane;
      const float m = rows(i);
      const DocRange range = walk.of(n);
      if (i0 >= most_begin && lo == hi && range.one() && range.lo == lo) {
        whole = fmaxf(whole, m);
        continue;
      }
      const int id = i < a.Lq ? d0[i] : -1;
      uint64_t left = __ballot(id >= lo && id <= hi);
      for (int run = 0; run < kLiftRuns && left != 0; ++run) {
        const int present = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        take(id == present ? m : 0.f, i0, doc == present);
        left &= ~__ballot(id == present);
      }
      for (; left != 0; left &= left - 1) {  // of ids in no order one by one
        const int r = __builtin_ctzll(left);
        const float one = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m), r));
        if (__builtin_amdgcn_readlane(id, r) == doc && i0 + r >= begin) top = fmaxf(top, one);
      }
    }
  }
  tops[wave][lane] = fmaxf(top, wave_reduce_max(whole));
  __syncthreads();
  if (wave != 0 || j >= a.Lk) return;
#pragma unroll
  for (int w = 0; w < kLiftWaves; ++w) top = w == 0 ? tops[0][lane] : fmaxf(top, tops[w][lane]);
  a.key_lift[bc * a.Lk + j] = grad_scale(ok ? top : 0.f);
}

void check_tensor(const torch::Tensor& x, const torch::Tensor& q, const char* name) {
  const int64_t per16 = 16 / x.element_size();
  TORCH_CHECK(x.is_cuda() && x.device() == q.device() && x.dim() == 4 && x.scalar_type() == q.scalar_type(),
              "attention: ", name, " is [batch, length, heads, width] of q's type on its device");
  TORCH_CHECK(x.size(0) == q.size(0) && x.size(3) == q.size(3), "attention: ", name, " does not fit q");
  TORCH_CHECK(x.stride(3) == 1 && x.stride(0) % per16 == 0 && x.stride(1) % per16 == 0 && x.stride(2) % per16 == 0 &&
                  reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0,
              "attention: rows of ", name, " begin at 16-byte borders");
  TORCH_CHECK(x.size(1) <= 1 || x.stride(1) * x.element_size() <= (1 << 24), "attention: rows of ", name, " lie over 16 MB apart");
}

RowStrides strides_of(const torch::Tensor& x) { return {x.stride(0), x.stride(1), x.stride(2)}; }

const int* ids(const c10::optional<torch::Tensor>& x, const torch::Tensor& q, std::vector<int64_t> shape, const char* name) {
  if (!x.has_value()) return nullptr;
  TORCH_CHECK(x->device() == q.device() && x->scalar_type() == at::kInt && x->is_contiguous() &&
                  x->sizes() == at::IntArrayRef(shape), "attention: ", name, " has another shape, type or device");
  return x->data_ptr<int>();
}

AttnArgs arguments(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v, double scale, double softcap,
                   const c10::optional<torch::Tensor>& slopes, bool causal, const c10::optional<torch::Tensor>& prefix,
                   const c10::optional<torch::Tensor>& q_doc, const c10::optional<torch::Tensor>& k_doc) {
  check_tensor(q, q, "q");
  check_tensor(k, q, "k");
  check_tensor(v, q, "v");
  const int64_t B = q.size(0), Lq = q.size(1), H = q.size(2), D = q.size(3), Lk = k.size(1), Hk = k.size(2);
  TORCH_CHECK(B > 0 && Lq > 0 && Lk > 0 && H > 0 && Hk > 0 && H % Hk == 0, "attention: empty, or heads that do not divide");
  TORCH_CHECK(D % 8 == 0 && D >= 8 && D <= 128, "attention: widths of 8 to 128 in steps of 8, got ", D);
  TORCH_CHECK(v.size(1) == Lk && v.size(2) == Hk, "attention: k and v differ");
  TORCH_CHECK(std::max(Lq, Lk) < (int64_t{1} << 30) && B * H < (int64_t{1} << 31) / 2 && q_doc.has_value() == k_doc.has_value(),
              "attention: too long, or documents of one side only");
  if (slopes.has_value())
    TORCH_CHECK(slopes->device() == q.device() && slopes->scalar_type() == at::kFloat && slopes->is_contiguous() &&
                    slopes->dim() == 1 && slopes->size(0) == H, "attention: slopes are fp32 [heads]");
  AttnArgs a{};
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr();
  a.qs = strides_of(q); a.ks = strides_of(k); a.vs = strides_of(v);
  a.B = B; a.Lq = Lq; a.Lk = Lk; a.H = H; a.Hk = Hk; a.D = D;
  a.scale = static_cast<float>(scale);
  a.softcap = static_cast<float>(softcap);
  a.slopes = slopes.has_value() ? slopes->data_ptr<float>() : nullptr;
  a.causal = causal;
  a.prefix = causal ? ids(prefix, q, {B}, "prefix") : nullptr;
  a.q_doc = ids(q_doc, q, {B, Lq}, "documents");
  a.k_doc = ids(k_doc, q, {B, Lk}, "key_documents");
  return a;
}

// The ids of every 64 rows, or nothing.
torch::Tensor doc_ranges(const c10::optional<torch::Tensor>& ids, int B, int L, hipStream_t stream) {
  if (!ids.has_value()) return torch::Tensor();
  const int tiles = (L + kDocTile - 1) / kDocTile;
  auto out = torch::empty({static_cast<int64_t>(B) * tiles, 4}, ids->options());
  TORCH_CHECK(launchable(static_cast<int64_t>(B) * tiles, WAVE), "attention: too many rows");
  doc_ranges_kernel<<<B * tiles, WAVE, 0, stream>>>(
      ids->data_ptr<int>(), L, tiles, reinterpret_cast<DocRange*>(out.data_ptr<int>()));
  HIP_CHECK_LAST();
  return out;
}

const DocRange* ranges_of(const torch::Tensor& x) {
  return x.defined() ? reinterpret_cast<const DocRange*>(x.data_ptr<int>()) : nullptr;
}

// The order of a side's blocks, or nothing where there is none to choose or so many that
// they even out by themselves.
torch::Tensor block_order(const torch::Tensor& own, int own_rows, const torch::Tensor& other, int other_rows, int B, hipStream_t stream) {
  const int blocks = (own_rows + kBlockRows - 1) / kBlockRows;
  if (!own.defined() || blocks < 2 || blocks > kMostOrdered || !launchable(B, kMostOrdered)) return torch::Tensor();
  auto out = torch::empty({B, blocks}, own.options());
  block_order_kernel<<<B, (blocks + WAVE - 1) / WAVE * WAVE, 0, stream>>>(
      ranges_of(own), (own_rows + kDocTile - 1) / kDocTile, ranges_of(other), (other_rows + kDocTile - 1) / kDocTile, blocks, out.data_ptr<int>());
  HIP_CHECK_LAST();
  return out;
}

const int* order_of(const torch::Tensor& x) { return x.defined() ? x.data_ptr<int>() : nullptr; }

// The ids of both sides by tiles; one tensor for both stays one.
struct Ranges {
  torch::Tensor k, q;
  Ranges(const AttnArgs& a, const c10::optional<torch::Tensor>& q_doc, const c10::optional<torch::Tensor>& k_doc, bool both, hipStream_t stream) {
    k = doc_ranges(k_doc, a.B, a.Lk, stream);
    if (both) q = a.q_doc == a.k_doc && a.Lq == a.Lk ? k : doc_ranges(q_doc, a.B, a.Lq, stream);
  }
};

}  // namespace

void key_lifts(const AttnArgs& a, const DocRange* q_ranges, hipStream_t stream) {
  const int key_tiles = (a.Lk + WAVE - 1) / WAVE;
  const int64_t blocks = static_cast<int64_t>(a.B) * a.Hk * key_tiles;
  TORCH_CHECK(launchable(blocks, kLiftWaves * WAVE), "attention: too many rows");
  key_lifts_kernel<<<blocks, kLiftWaves * WAVE, 0, stream>>>(a, q_ranges, key_tiles);
  HIP_CHECK_LAST();
}

// {o [B, Lq, H, D], lse [B, H, Lq], what rounding took from o (16-bit types, if `keep_rest`) or nothing}
std::vector<torch::Tensor> attention_fwd(torch::Tensor q, torch::Tensor k, torch::Tensor v, double scale, double softcap,
                                         c10::optional<torch::Tensor> slopes, bool causal,
                                         c10::optional<torch::Tensor> prefix, c10::optional<torch::Tensor> q_doc,
                                         c10::optional<torch::Tensor> k_doc, bool keep_rest) {
  AttnArgs a = arguments(q, k, v, scale, softcap, slopes, causal, prefix, q_doc, k_doc);
  at::DeviceGuard guard(q.device());
  auto o = torch::empty({a.B, a.Lq, a.H, a.D}, q.options());
  keep_rest = keep_rest && q.scalar_type() != at::kFloat;
  auto rest = torch::empty(keep_rest ? o.sizes() : at::IntArrayRef({0}), q.options());
  a.o_rest = keep_rest ? rest.data_ptr() : nullptr;
  auto lse = torch::empty({a.B, a.H, a.Lq}, q.options().dtype(at::kFloat));
  a.o = o.data_ptr();
  a.lse = lse.data_ptr<float>();
  auto stream = at::hip::getCurrentHIPStream();
  const bool ordered = attention_in_tiles(a) && a.Lq > kBlockRows;
  const Ranges ranges(a, q_doc, k_doc, ordered, stream);
  const auto order = ordered ? block_order(ranges.q, a.Lq, ranges.k, a.Lk, a.B, stream) : torch::Tensor();
  a.q_order = order_of(order);
  DISPATCH_FLOAT(q.scalar_type(), "attention", [&] { attention_forward<T>(a, ranges_of(ranges.k), q.options(), stream); });
  HIP_CHECK_LAST();
  return {o, lse, rest};
}

// {dq, dk, dv}, contiguous
std::vector<torch::Tensor> attention_bwd(torch::Tensor dout, torch::Tensor q, torch::Tensor k, torch::Tensor v,
                                         torch::Tensor o, torch::Tensor lse, torch::Tensor rest, double scale, double softcap,
                                         c10::optional<torch::Tensor> slopes, bool causal,
                                         c10::optional<torch::Tensor> prefix, c10::optional<torch::Tensor> q_doc,
                                         c10::optional<torch::Tensor> k_doc) {
  AttnArgs a = arguments(q, k, v, scale, softcap, slopes, causal, prefix, q_doc, k_doc);
  check_tensor(dout, q, "the gradient");
  TORCH_CHECK(dout.sizes() == q.sizes() && o.sizes() == q.sizes() && o.is_contiguous() && o.scalar_type() == q.scalar_type() &&
                  lse.numel() == static_cast<int64_t>(a.B) * a.H * a.Lq && lse.is_contiguous() && lse.scalar_type() == at::kFloat);
  at::DeviceGuard guard(q.device());
  auto dq = torch::empty({a.B, a.Lq, a.H, a.D}, q.options());
  auto dk = torch::empty({a.B, a.Lk, a.Hk, a.D}, q.options());
  auto dv = torch::empty({a.B, a.Lk, a.Hk, a.D}, q.options());
  auto delta = torch::empty({a.B, a.H, a.Lq}, lse.options());
  TORCH_CHECK(rest.numel() == 0 || (rest.sizes() == o.sizes() && rest.is_contiguous() && rest.scalar_type() == o.scalar_type()));
  a.o = o.data_ptr(); a.lse = lse.data_ptr<float>();
  a.o_rest = rest.numel() > 0 ? rest.data_ptr() : nullptr;
  a.dout = dout.data_ptr(); a.gs = strides_of(dout);
  a.delta = delta.data_ptr<float>();
  a.dq = dq.data_ptr(); a.dk = dk.data_ptr(); a.dv = dv.data_ptr();
  auto stream = at::hip::getCurrentHIPStream();
  const Ranges ranges(a, q_doc, k_doc, true, stream);
  const bool one = ranges.q.is_same(ranges.k);
  const auto q_order = block_order(ranges.q, a.Lq, ranges.k, a.Lk, a.B, stream);
  const auto k_order = one ? q_order : block_order(ranges.k, a.Lk, ranges.q, a.Lq, a.B, stream);
  a.q_order = order_of(q_order);
  a.k_order = order_of(k_order);
  torch::Tensor tops;  // of rows, blocks and keys, one behind another
  if (q.scalar_type() == at::kHalf) {
    const int64_t heads = static_cast<int64_t>(a.B) * a.H, blocks = heads * ((a.Lq + 31) / 32);
    tops = torch::empty({heads * a.Lq + blocks + static_cast<int64_t>(a.B) * a.Hk * a.Lk}, lse.options());
    a.row_top = tops.data_ptr<float>();
    a.block_top = a.row_top + heads * a.Lq;
    a.key_lift = a.block_top + blocks;
  }
  DISPATCH_FLOAT(q.scalar_type(), "attention", [&] {
    attention_backward<T>(a, ranges_of(ranges.k), ranges_of(ranges.q), q.options(), stream);
  });
  HIP_CHECK_LAST();
  return {dq, dk, dv};
}
