// The paged 4-bit cache (paged4.cuh) besides appending and attention: reading values back, and eviction by received weight.
//
// Eviction keeps, for each sequence of more than `budget` tokens and each KV head by itself, the last `recent` tokens and of
// the others the budget - recent of largest mass, ties to the lower slot, and moves them, in order, to slots 0 .. budget - 1.
//
// select: a cluster of CTAs per (sequence, head) finds the least kept mass by radix: 11, 11 and 10 bits of the weights' order
// as whole numbers, each pass a histogram in shared memory that the cluster's CTAs add up through distributed shared
// memory.  A thread holds the 16 slots of a block, in order, so a scan of the threads' counts gives each kept slot its place.
// move: 8 lanes per token copy its codes, parameters and mass.  To other pages in one pass; in place through a packed
// copy, since the kept tokens' places overlap.
#include "paged4.cuh"

#include <cooperative_groups.h>

namespace mamf {
namespace kv4 {

using namespace paged4;
namespace cg = cooperative_groups;

__device__ int g_err = 0;
__device__ __forceinline__ void record(int code) { atomicCAS(&g_err, 0, code); }

// ---- read ------------------------------------------------------------------------------------------
constexpr int NR = 256;

template <typename T> __device__ __forceinline__ void store8(T* p, const float* f) {
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8 / N; ++i) {
    Vec16<T> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v.v[j] = from_f<T>(f[i * N + j]);
    st16(p + i * N, v);
  }
}
// 8 dims of a word of codes
__device__ __forceinline__ void values8(uint32_t w, uint32_t params, const Base& base, float* f) {
  uint32_t h[4];
  decode(w, levels_of(params, base), base, h);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
    f[e] = v.x;
    f[e + 4] = v.y;
  }
}

// TPT lanes per token, of every gridDim.y-th head: 8 dims of each half of keys and values a lane.
template <typename T, int HD>
__global__ void __launch_bounds__(NR) read_kernel(const Cache4 c, T* __restrict__ k, T* __restrict__ v) {
  constexpr int TPT = HD / 16, J = HD / 32;
  if (blockIdx.x + blockIdx.y == 0)
    for (int b = threadIdx.x; b < c.B; b += NR)
      if (!in_order(c, b)) record(ERR_LENGTH);
  const int sub = threadIdx.x % TPT, d = sub * 8;
  const int64_t item = ((int64_t)blockIdx.x * NR + threadIdx.x) / TPT;
  if (item >= c.T) return;
  const int t = (int)item, b = sequence_of(c.cu, c.B, t);
  int slot = 0, pg = -1;
  if (b >= 0) {
    const int t0 = c.cu[b], n = c.cu[b + 1] - t0, len = c.lens[b];
    slot = len - n + (t - t0);
    if (in_order(c, b) && t >= t0 && t - t0 < n && len >= 0) {
      if (slot >= 0) {                                // a sequence of fewer tokens than were asked for: zeros in front
        const int j = slot >> c.shift;
        pg = j < c.W ? c.table[(int64_t)b * c.W + j] : -1;
        if (pg < 0 || pg >= c.P) { pg = -1; if (sub == 0) record(ERR_PAGE); }
      }
    } else if (sub == 0) {
      record(ERR_LENGTH);
    }
  }
  for (int g = blockIdx.y; g < c.G; g += gridDim.y) {
    float f[32] = {};
    if (pg >= 0) {
      const uint8_t* blk = block_of<HD>(c, pg, g, slot);
      const int row = slot & 15;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint8_t* at = blk + x * HALF<HD>;
        const uint32_t w0 = *reinterpret_cast<const uint32_t*>(at + row * (HD / 2) + sub * 4);
        const uint32_t w1 = *reinterpret_cast<const uint32_t*>(at + row * (HD / 2) + HD / 4 + sub * 4);
        const uint32_t params = *reinterpret_cast<const uint32_t*>(at + PARAMS<HD> + (row * (J / 2) + sub % (J / 2)) * 4);
        values8(w0, params, c.base, f + 16 * x);
        values8(w1, params, c.base, f + 16 * x + 8);
      }
    }
    const int64_t to = ((int64_t)t * c.G + g) * HD + d;
    store8(k + to, f);
    store8(k + to + HD / 2, f + 8);
    store8(v + to, f + 16);
    store8(v + to + HD / 2, f + 24);
  }
}

// ---- eviction: which slots -------------------------------------------------------------------------
constexpr int NS = 512, KPT = 16, BINS = 2048;       // threads, slots of a thread, bins of a pass
constexpr int MOST = 8;                               // CTAs of a cluster

struct Evict {
  Cache4 c;
  const int* out_table;
  int* kept;                                          // (B, G, budget)
  int* lens_out;                                      // (B)
  uint8_t* packed;                                    // in place: the kept tokens on their way
  int out_W, budget, recent;
};

// The order of floats as that of whole numbers, -0 as 0
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sums of (a, b) over the threads before this one, and over all.
__device__ __forceinline__ int2 scan2(int2 v, int2& total, int2* sm) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int2 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, x.x, o), b = __shfl_up_sync(0xffffffffu, x.y, o);
    if (lane >= o) { x.x += a; x.y += b; }
  }
  if (lane == 31) sm[w] = x;
  __syncthreads();
  int2 before = make_int2(0, 0);
  total = make_int2(0, 0);
#pragma unroll
  for (int i = 0; i < NS / 32; ++i) {
    if (i < w) { before.x += sm[i].x; before.y += sm[i].y; }
    total.x += sm[i].x;
    total.y += sm[i].y;
  }
  __syncthreads();
  return make_int2(before.x + x.x - v.x, before.y + x.y - v.y);
}

__global__ void __launch_bounds__(NS) select_kernel(const Evict p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  __shared__ int hist[2][BINS];                       // the passes take turns
  __shared__ int2 sm[NS / 32], mine;
  __shared__ int s_bin, s_above;
  const Cache4& c = p.c;
  const int g = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int len = cached_length(c, c.lens[b]), K = p.budget;
  int* kept = p.kept + ((int64_t)b * c.G + g) * K;
  if (g == 0 && rank == 0 && tid == 0) {
    p.lens_out[b] = min(len, K);
    if (len != c.lens[b]) record(ERR_LENGTH);
  }
  if (len <= K) {                                     // the cluster's CTAs agree on this: nobody waits
    for (int i = rank * NS + tid; i < K; i += C * NS) kept[i] = i < len ? i : -1;
    return;
  }
  const int old = len - p.recent;                     // the slots that compete for `want` places
  int want = K - p.recent;
  // batch i of this CTA: slots (i C + rank) NS KPT + tid KPT ..
  const int batches = (int)(((int64_t)old + (int64_t)C * NS * KPT - 1) / ((int64_t)C * NS * KPT));
  uint32_t key[KPT];
  auto first_of = [&](int i) { return (int64_t)(i * C + rank) * (NS * KPT) + tid * KPT; };
  auto load = [&](int i) {
    const int64_t s0 = first_of(i);
    int pg = -1;
    if (s0 < old) {
      pg = c.table[(int64_t)b * c.W + (s0 >> c.shift)];
      if (pg < 0 || pg >= c.P) { pg = -1; record(ERR_PAGE); }
    }
    const float* m = c.mass + (((int64_t)pg * c.G + g) << c.shift) + (s0 & (c.page - 1));
#pragma unroll
    for (int e = 0; e < KPT; e += 4) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (pg >= 0) v = *reinterpret_cast<const float4*>(m + e);
      key[e] = order_of(v.x);
      key[e + 1] = order_of(v.y);
      key[e + 2] = order_of(v.z);
      key[e + 3] = order_of(v.w);
    }
  };
  load(0);
  uint32_t at = 0;                                    // the bits of the least kept weight found so far
  for (int i = tid; i < 2 * BINS; i += NS) (&hist[0][0])[i] = 0;
  __syncthreads();
  int shift = 32;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass < 2 ? 11 : 10;
    const uint32_t above = pass == 0 ? 0u : 0xFFFFFFFFu << shift;      // bits that are settled
    shift -= bits;
    int* h = hist[pass & 1];
    if (want > 0)
#pragma unroll 1
      for (int i = 0; i < batches; ++i) {
        if (batches > 1) load(i);
        const int64_t s0 = first_of(i);
#pragma unroll
        for (int e = 0; e < KPT; ++e)
          if (s0 + e < old && (key[e] & above) == at) atomicAdd(&h[key[e] >> shift & ((1 << bits) - 1)], 1);
      }
    cluster.sync();
    // bins from the top: thread t takes BINS / NS of them, the highest first
    constexpr int PER = BINS / NS;
    int n[PER], sum = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int bin = BINS - 1 - (tid * PER + e);
      n[e] = 0;
      for (int r = 0; r < C; ++r) n[e] += *cluster.map_shared_rank(&h[bin], r);
      sum += n[e];
    }
    int2 total;
    int before = scan2(make_int2(sum, 0), total, sm).x;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (before < want && want <= before + n[e]) { s_bin = BINS - 1 - (tid * PER + e); s_above = before; }
      before += n[e];
    }
    if (want == 0 && tid == 0) { s_bin = (1 << bits) - 1; s_above = 0; }      // no place: nothing is as heavy
    __syncthreads();
    at |= (uint32_t)s_bin << shift;
    want -= s_above;
    cluster.sync();                                   // everybody has read this pass's bins
    if (pass == 0) {                                  // for the third pass
      for (int i = tid; i < BINS; i += NS) h[i] = 0;
      __syncthreads();
    }
  }
  // `want` of those as heavy as `at` are kept, the lowest slots, and all heavier ones
  int2 done = make_int2(0, 0);                        // heavier, and as heavy, in slots before the batch
#pragma unroll 1
  for (int i = 0; i < batches; ++i) {
    if (batches > 1) load(i);
    const int64_t s0 = first_of(i);
    int2 v = make_int2(0, 0), total;
#pragma unroll
    for (int e = 0; e < KPT; ++e)
      if (s0 + e < old) { v.x += key[e] > at; v.y += key[e] == at; }
    int2 x = scan2(v, total, sm);
    if (tid == 0) mine = total;
    cluster.sync();
    int2 batch = make_int2(0, 0);
    for (int r = 0; r < C; ++r) {
      const int2 o = *cluster.map_shared_rank(&mine, r);
      if (r < rank) { x.x += o.x; x.y += o.y; }
      batch.x += o.x;
      batch.y += o.y;
    }
    x.x += done.x;
    x.y += done.y;
    done.x += batch.x;
    done.y += batch.y;
#pragma unroll
    for (int e = 0; e < KPT; ++e)
      if (s0 + e < old) {
        const bool heavier = key[e] > at, same = key[e] == at;
        if (heavier || (same && x.y < want)) kept[x.x + min(x.y, want)] = (int)(s0 + e);
        x.x += heavier;
        x.y += same;
      }
    cluster.sync();                                   // everybody has read `mine`
  }
  for (int i = rank * NS + tid; i < p.recent; i += C * NS) kept[K - p.recent + i] = old + i;
}

// ---- eviction: the move ----------------------------------------------------------------------------
constexpr int NM = 256, LANES = 8, UNROLL = 4;
template <int HD> constexpr int RECORD = HD + HD / 8 + 16;          // a packed token: codes, parameters, mass

enum Mode { DIRECT, PACK, UNPACK };

// A token's pieces by lane: lanes 0-3 keys, 4-7 values, 16 bytes of codes each (8 of 64 dims); lanes 0 and 4 the
// parameters; lane 1 the mass.
template <int HD> struct Piece {
  uint4 code;
  uint2 param;
  float mass;
};
template <int HD>
__device__ __forceinline__ void get(Piece<HD>& x, const uint8_t* half, int row, int q, const float* mass, int lane) {
  if (HD == 128) x.code = *reinterpret_cast<const uint4*>(half + row * (HD / 2) + q * 16);
  else *reinterpret_cast<uint2*>(&x.code) = *reinterpret_cast<const uint2*>(half + row * (HD / 2) + q * 8);
  if (q == 0) {
    if (HD == 128) x.param = *reinterpret_cast<const uint2*>(half + PARAMS<HD> + row * (HD / 16));
    else x.param.x = *reinterpret_cast<const uint32_t*>(half + PARAMS<HD> + row * (HD / 16));
  }
  if (lane == 1) x.mass = *mass;
}
template <int HD>
__device__ __forceinline__ void put(const Piece<HD>& x, uint8_t* half, int row, int q, float* mass, int lane) {
  if (HD == 128) *reinterpret_cast<uint4*>(half + row * (HD / 2) + q * 16) = x.code;
  else *reinterpret_cast<uint2*>(half + row * (HD / 2) + q * 8) = *reinterpret_cast<const uint2*>(&x.code);
  if (q == 0) {
    if (HD == 128) *reinterpret_cast<uint2*>(half + PARAMS<HD> + row * (HD / 16)) = x.param;
    else *reinterpret_cast<uint32_t*>(half + PARAMS<HD> + row * (HD / 16)) = x.param.x;
  }
  if (lane == 1) *mass = x.mass;
}

template <int HD, int MODE>
__global__ void __launch_bounds__(NM) move_kernel(const Evict p) {
  const Cache4& c = p.c;
  const int lane = threadIdx.x % LANES, q = lane & 3, side = lane >> 2;
  const int g = blockIdx.y, b = blockIdx.z;
  const int64_t row0 = ((int64_t)b * c.G + g) * p.budget;
  const int* table = c.table + (int64_t)b * c.W;
  const int* to = p.out_table + (int64_t)b * p.out_W;
  constexpr int GROUPS = NM / LANES;
  const int r0 = blockIdx.x * (GROUPS * UNROLL) + threadIdx.x / LANES;
  int src[UNROLL];
  uint8_t* dst[UNROLL];
  float* dst_mass[UNROLL];
  Piece<HD> x[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int r = r0 + u * GROUPS;
    src[u] = r < p.budget ? p.kept[row0 + r] : -1;
    if (MODE != DIRECT && src[u] == r) src[u] = -1;   // it stays
    dst[u] = nullptr;
    if (src[u] < 0) continue;
    if (MODE == PACK) {
      dst[u] = p.packed + (row0 + r) * RECORD<HD>;
      continue;
    }
    const int pg = to[r >> c.shift];
    if (pg >= 0 && pg < c.P) {
      dst[u] = block_of<HD>(c, pg, g, r) + side * HALF<HD>;
      dst_mass[u] = c.mass + (((int64_t)pg * c.G + g) << c.shift) + (r & (c.page - 1));
    } else if (lane == 0) {
      record(ERR_PAGE);
    }
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    if (!dst[u]) continue;
    const int r = r0 + u * GROUPS;
    if (MODE == UNPACK) {
      const uint8_t* rec = p.packed + (row0 + r) * RECORD<HD>;
      if (HD == 128) x[u].code = *reinterpret_cast<const uint4*>(rec + lane * 16);
      else *reinterpret_cast<uint2*>(&x[u].code) = *reinterpret_cast<const uint2*>(rec + lane * 8);
      x[u].param = *reinterpret_cast<const uint2*>(rec + HD + side * 8);
      x[u].mass = *reinterpret_cast<const float*>(rec + HD + 16);
      continue;
    }
    const int pg = table[src[u] >> c.shift];
    if (pg < 0 || pg >= c.P) { dst[u] = nullptr; if (lane == 0) record(ERR_PAGE); continue; }
    get<HD>(x[u], block_of<HD>(c, pg, g, src[u]) + side * HALF<HD>, src[u] & 15, q,
            c.mass + (((int64_t)pg * c.G + g) << c.shift) + (src[u] & (c.page - 1)), lane);
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    if (!dst[u]) continue;
    const int r = r0 + u * GROUPS;
    if (MODE == PACK) {
      if (HD == 128) *reinterpret_cast<uint4*>(dst[u] + lane * 16) = x[u].code;
      else *reinterpret_cast<uint2*>(dst[u] + lane * 8) = *reinterpret_cast<const uint2*>(&x[u].code);
      if (q == 0) *reinterpret_cast<uint2*>(dst[u] + HD + side * 8) = x[u].param;
      if (lane == 1) *reinterpret_cast<float*>(dst[u] + HD + 16) = x[u].mass;
    } else {
      put<HD>(x[u], dst[u], r & 15, q, dst_mass[u], lane);
    }
  }
}

template <int HD> void launch_move(Evict& p, bool in_place) {
  const dim3 grid((unsigned)((p.budget + NM / LANES * UNROLL - 1) / (NM / LANES * UNROLL)), (unsigned)p.c.G, (unsigned)p.c.B);
  if (!in_place) { move_kernel<HD, DIRECT><<<grid, NM, 0, stream()>>>(p); MAMF_LAUNCH_CHECK(); return; }
  const at::Tensor ws = at::empty({(int64_t)p.c.B * p.c.G * p.budget * RECORD<HD>}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA));
  p.packed = ws.data_ptr<uint8_t>();
  move_kernel<HD, PACK><<<grid, NM, 0, stream()>>>(p);
  MAMF_LAUNCH_CHECK();
  move_kernel<HD, UNPACK><<<grid, NM, 0, stream()>>>(p);
  MAMF_LAUNCH_CHECK();
}

}  // namespace kv4

// Values of the last cu[b + 1] - cu[b] tokens of each sequence: k, v (T, G, hd).
std::vector<at::Tensor> kv4_read(at::Tensor blocks, at::Tensor table, at::Tensor cu, at::Tensor lens, int64_t T, at::ScalarType dtype) {
  using namespace kv4;
  TORCH_CHECK(blocks.is_cuda() && blocks.dim() == 4, "kv_read: blocks (P, G, page / 16, 18 hd) on a GPU");
  c10::cuda::CUDAGuard guard(blocks.device());
  TORCH_CHECK(T >= 0, "kv_read: tokens must not be negative");
  const int64_t hd = blocks.size(3) / 18;
  const Cache4 c = check_cache4("kv_read", blocks, c10::nullopt, table, &cu, lens, T, hd);
  const auto opts = blocks.options().dtype(dtype);
  std::vector<at::Tensor> out{at::empty({T, c.G, hd}, opts), at::empty({T, c.G, hd}, opts)};
  if (T == 0) return out;
  if (c.B == 0) { out[0].zero_(); out[1].zero_(); return out; }
  const int64_t units = (T * (hd / 16) + NR - 1) / NR;
  TORCH_CHECK(units < (1LL << 31), "kv_read: sizes");
  const dim3 grid((unsigned)units, (unsigned)std::max<int64_t>(1, std::min<int64_t>(c.G, 8LL * num_sms() / units)));
  MAMF_DISPATCH_FLOAT_BF16(dtype, "kv_read", [&] {
    auto* k = (scalar_t*)out[0].data_ptr();
    auto* v = (scalar_t*)out[1].data_ptr();
    if (hd == 128) read_kernel<scalar_t, 128><<<grid, NR, 0, stream()>>>(c, k, v);
    else read_kernel<scalar_t, 64><<<grid, NR, 0, stream()>>>(c, k, v);
  });
  MAMF_LAUNCH_CHECK();
  return out;
}

// Moves the kept tokens (out_table: to its pages; none: in place).  Returns the kept slots (B, G, budget), -1 for none, and
// the new lengths.
std::vector<at::Tensor> kv4_evict(at::Tensor blocks, at::Tensor mass, at::Tensor table, at::Tensor lens, int64_t budget,
                                  int64_t recent, c10::optional<at::Tensor> out_table) {
  using namespace kv4;
  TORCH_CHECK(blocks.is_cuda() && blocks.dim() == 4, "kv_evict: blocks (P, G, page / 16, 18 hd) on a GPU");
  c10::cuda::CUDAGuard guard(blocks.device());
  const int64_t hd = blocks.size(3) / 18;
  Evict p{};
  p.c = check_cache4("kv_evict", blocks, mass, table, nullptr, lens, 0, hd);
  TORCH_CHECK(aligned16(p.c.mass), "kv_evict: 16-byte aligned mass");
  TORCH_CHECK(budget >= 1 && recent >= 0 && recent <= budget && budget < (1LL << 30), "kv_evict: 0 <= recent <= budget and budget >= 1, got ",
              recent, " and ", budget);
  const at::Tensor& to = out_table.has_value() ? *out_table : table;
  TORCH_CHECK(to.is_cuda() && to.device() == blocks.device() && to.is_contiguous() && to.scalar_type() == at::kInt && to.dim() == 2 &&
              to.size(0) == p.c.B, "kv_evict: a contiguous int32 out_table with a row for each sequence");
  const int64_t most = std::min<int64_t>(budget, (int64_t)p.c.W * p.c.page);      // tokens that a sequence can keep
  TORCH_CHECK(to.size(1) * p.c.page >= most, "kv_evict: out_table has room for ", to.size(1) * p.c.page, " of ", most, " tokens");
  TORCH_CHECK(p.c.B < 65536, "kv_evict: at most 65535 sequences");
  at::Tensor kept = at::empty({p.c.B, p.c.G, budget}, table.options()), lens_out = at::empty({p.c.B}, table.options());
  if (p.c.B == 0) return {kept, lens_out};
  p.out_table = to.data_ptr<int>();
  p.out_W = (int)to.size(1);
  p.kept = kept.data_ptr<int>();
  p.lens_out = lens_out.data_ptr<int>();
  p.budget = (int)budget;
  p.recent = (int)recent;
  // CTAs per (sequence, head): as many as the table's longest sequence fills, up to a cluster
  int C = 1;
  while (C < MOST && (int64_t)C * NS * KPT < (int64_t)p.c.W * p.c.page) C *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)C, (unsigned)p.c.G, (unsigned)p.c.B);
  cfg.blockDim = dim3(NS);
  cfg.stream = stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  MAMF_CUDA_CHECK(cudaLaunchKernelEx(&cfg, select_kernel, p));
  const bool in_place = to.data_ptr() == table.data_ptr();
  if (hd == 128) launch_move<128>(p, in_place); else launch_move<64>(p, in_place);
  return {kept, lens_out};
}

int64_t kv4_error(bool clear) { return paged::take_code(kv4::g_err, clear); }

}  // namespace mamf
