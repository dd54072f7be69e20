// Causal attention of a step's prompt rows over the 4-bit cache (kv4.h): fresh prompts and chunks that continue one.
//
// A workgroup of 4 waves has 32 query rows of each of GH heads of one kv head (GH = 4: 32 rows of the 128-row work item, 2: 64,
// 1: 128).  Keys and values advance in tiles of 64 tokens: a thread loads a quarter row of K and of V (D / 8 bytes each) while
// the tile before it computes, widens them and writes them to LDS as T.  So a tile is widened once for 128 rows of queries:
// 32 conversions a wave beside the 32 MFMAs of 32 cycles that it feeds (D = 128).
//
// v_mfma_f32_32x32x16: S^T = K Q^T and O^T = V^T P^T, so that a query is a lane's column in every accumulator: its maximum
// and sum are the lane's own (and its partner's, lane ^ 32), and S^T's accumulator, packed, is the B operand of the second product.
// V's rows become columns by the transposing LDS read.
//
// Z > 1: few rows after long contexts leave CUs idle, so that Z workgroups share an item's tiles; each leaves its rows' maximum,
// sum and unnormalised result, which kv4_prefill_merge_kernel joins.
//
// 4 x 4096 rows of 32 / 8 heads of 128 take 508 us (1.05 PFLOP/s; a large matrix product reaches 1.40): the matrix cores work in half
// of a CU's busy cycles at 2.0 GHz, vector instructions issue in 48 %, a wave's own products and softmax one after the other.  Scores of the
// next tile beside this one's softmax need 32 registers more, which the compiler takes from elsewhere: with 64 keys at a time
// they spill (1320 us), with 32 keys it is 678 us, and 760 with the order prescribed.
#include "common.h"
#include "kv4.h"
#include "device.h"
#include "launch.h"

namespace kgc {

constexpr int KV4_BM = 128, KV4_BN = 64;

__device__ __forceinline__ float kv4_max_pair(float x) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <typename T, int D, int GH, int BUFS>
__global__ __launch_bounds__(256, BUFS == 2 ? 2 : D == 128 ? 3 : 4) void kv4_prefill_kernel(
    const T* __restrict__ q, T* __restrict__ out, const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
    const int* __restrict__ block_tables, int bt_stride, const int* __restrict__ qsl, const int* __restrict__ seq_lens,
    const int* __restrict__ work_seq, const int* __restrict__ work_mblk, int nq, int nkv, int bs_log2, float scale_log2,
    int num_blocks, int seqs, int rows_all, float* __restrict__ part_o, float* __restrict__ part_ml, int Z) {
  typedef typename Vec8<T>::type V8;
  constexpr int QB = KV4_BM / GH;                    // query rows of a workgroup
  constexpr int KS = D / 16, DT = D / 32, W = D / 32; // W: words of a thread's quarter row
  // Rows of the LDS tiles, padded: of K, 16 rows' same chunk touches all banks, of V, four rows' 32 bytes.  (Chunks swizzled
  // instead halve the conflicts, 40 % of the LDS's busy cycles; the exclusive ors cost more.)
  constexpr int KST = D + 8, VST = D + 16;
  __shared__ __attribute__((aligned(16))) T lds_k[BUFS][KV4_BN * KST], lds_v[BUFS][KV4_BN * VST];
  // The list's items have most keys first, and so have their blocks here; neighbours, which XCDs take in turn, are the head
  // groups, so that with a multiple of 8 of them an XCD's cache has one group's pages.
  const int G = nq / nkv, groups = nkv * (G / GH), rest = blockIdx.x / groups, group = blockIdx.x % groups;
  const int slice = rest % Z, sub = GH - 1 - rest / Z % GH, item = rest / Z / GH;
  const int seq = work_seq[item], mb = work_mblk[item];
  const int h = group / (G / GH), head0 = h * G + group % (G / GH) * GH;
  if (seq < 0 || seq >= seqs || mb < 0) return;        // the whole workgroup, and so below
  const int q0 = qsl[seq], q1 = qsl[seq + 1];
  int L_in = seq_lens[seq];
  KGC_DCHECK_RANGE(L_in, 0, (bt_stride << bs_log2) + 1, "prefill seq_len");
  const int L = min(L_in, bt_stride << bs_log2);
  // (compared before they are subtracted or multiplied: no difference or product of numbers that are none wraps)
  if (q0 < 0 || q1 <= q0 || q1 > rows_all || L < q1 - q0 || mb > (q1 - q0 - 1) / KV4_BM) return;
  const int qlen = q1 - q0, ctx0 = L - qlen, qbase = mb * KV4_BM + sub * QB;
  if (qbase >= qlen) return;
  const int* bt = block_tables + (int64_t)seq * bt_stride;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 31, hi = lane >> 5;
  const int bs = 1 << bs_log2, bsm = bs - 1;
  const int64_t page_bytes = kv4_page_bytes(bs, D);
  const int wrow = qbase + wave / GH * 32, head = head0 + wave % GH;
  const int all = (ctx0 + min(qbase + QB, qlen) - 1) / KV4_BN + 1;
  const int first = (int)((int64_t)all * slice / Z), tiles = (int)((int64_t)all * (slice + 1) / Z);   // [first, tiles)
  // no row of this wave sees further (it may have none)
  const int wave_tiles = wrow < qlen ? (ctx0 + min(wrow + 32, qlen) - 1) / KV4_BN + 1 : 0;

  // A wave loads 16 tokens of a tile, which lie in one page; tokens behind the last one are that one again, and masked.
  const int tok = tid >> 2, part = tid & 3;
  const int wv = __builtin_amdgcn_readfirstlane(wave);
  uint32_t kw[W], vw[W];
  uint8_t ks, vs;
  auto base_of = [&](int kt) { return min(kt * KV4_BN + 16 * wv, (L - 1) & ~15); };
  auto page_of = [&](int kt) { return kv4_page(bt, base_of(kt) >> bs_log2, bt_stride, num_blocks); };
  auto load = [&](int kt, int pg) {
    const int base = base_of(kt);
    const int64_t page = ((int64_t)pg * nkv + h) * page_bytes + (base & bsm) * (D / 2);
    const int64_t scales = ((int64_t)pg * nkv + h) * page_bytes + bs * (D / 2) + (base & bsm) * (D / 32);
    const int row = min(lane >> 2, L - 1 - base);
    const uint32_t at = row * (D / 2) + part * (D / 8), sc = row * (D / 32) + (part * D / 4) / 32;
    if constexpr (W == 4) {
      const u32x4 x = *reinterpret_cast<const u32x4*>((kc + page) + at), y = *reinterpret_cast<const u32x4*>((vc + page) + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) { kw[i] = x[i]; vw[i] = y[i]; }
    } else {
      const u32x2 x = *reinterpret_cast<const u32x2*>((kc + page) + at), y = *reinterpret_cast<const u32x2*>((vc + page) + at);
#pragma unroll
      for (int i = 0; i < 2; ++i) { kw[i] = x[i]; vw[i] = y[i]; }
    }
    ks = (kc + scales)[sc];
    vs = (vc + scales)[sc];
  };
  auto store = [&](int buf) {
    const float a = kv4_scale(ks), b = kv4_scale(vs);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      *reinterpret_cast<u32x4*>(&lds_k[buf][tok * KST + part * (D / 4) + 8 * i]) = fp4x8_widen<T>(kw[i], a);
      *reinterpret_cast<u32x4*>(&lds_v[buf][tok * VST + part * (D / 4) + 8 * i]) = fp4x8_widen<T>(vw[i], b);
    }
  };

  // Lane (row col, hi) has elements 16 s + 8 hi .. + 7; rows behind the prompt's last one are that one again, not stored
  const int qi = min(wrow + col, qlen - 1), qpos = ctx0 + qi;
  Pack8<T> qf[KS];
  const T* qrow = q + ((int64_t)(q0 + qi) * nq + head) * D + 8 * hi;
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s].u = *reinterpret_cast<const u32x4*>(qrow + 16 * s);
  int pg = page_of(first);                             // (an empty slice: a tile that is there, not used)
  load(first, pg);
  pg = page_of(first + 1);
  store(0);
  // q is there before the loop: a wait for it in there would be one for the next tile's loads, too
#pragma unroll
  for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[s].u));
  __syncthreads();
  f32x16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int kt = first; kt < tiles; ++kt) {
    if (kt + 1 < tiles) {
      load(kt + 1, pg);
      pg = page_of(kt + 2);
    }
    if (kt < wave_tiles) {
      const T* K = lds_k[BUFS == 2 ? kt - first & 1 : 0];
      const T* V = lds_v[BUFS == 2 ? kt - first & 1 : 0];
      f32x16 s[2];
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[g][i] = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          Pack8<T> kf;
          kf.u = *reinterpret_cast<const u32x4*>(K + (32 * g + col) * KST + 16 * j + 8 * hi);
          s[g] = mfma32x32x16(kf.v, qf[j].v, s[g]);
        }
      const int key0 = kt * KV4_BN + 4 * hi;           // element i of half g: key0 + 32 g + 8 (i / 4) + i % 4
      if (kt * KV4_BN + KV4_BN - 1 > ctx0 + wrow) {    // some row of the wave does not see all of the tile
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (key0 + 32 * g + 8 * (i >> 2) + (i & 3) > qpos) s[g][i] = -INFINITY;
      }
      // scores are scaled behind their maximum and their mask: the scale is above zero (the host refuses others)
      float top = s[0][0];
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = __builtin_elementwise_maximum(top, s[g][i]);   // (fmaxf quiets every score first)
      top = kv4_max_pair(top) * scale_log2;
      // the maximum moves only where it grows by more than 8: probabilities are then at most 2^8, and O is seldom rescaled
      if (__any(top > m + 8.f)) {
        const float to = fmaxf(m, top), f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= f;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] *= f;
      }
      const float ref = m == -INFINITY ? 0.f : m;
      V8 pf[4];
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          Pack8<T> p;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            // at most 2^8, rounded to T for the product; the sum, in 32 bits, is that of the rounded ones
            p.h[i] = from_f<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[g][8 * j + i], scale_log2, -ref)));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) l = kv4_add_pair<T>(p.u[i], l);
          pf[2 * g + j] = p.v;
        }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          const T* src = V + (16 * j + 4 * hi + ((lane & 15) >> 2)) * VST + 32 * t + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
          const u32x2 a = ld_tr4(src), b = ld_tr4(src + 8 * VST);
          Pack8<T> vf;
          vf.u = u32x4{a.x, a.y, b.x, b.y};
          o[t] = mfma32x32x16(vf.v, pf[j], o[t]);
        }
    }
    if (kt + 1 < tiles) {
      if constexpr (BUFS == 1) __syncthreads();
      store(BUFS == 2 ? kt - first + 1 & 1 : 0);
      __syncthreads();
    }
  }
  l += __shfl_xor(l, 32, 64);
  if (Z > 1) {
    if (wrow + col >= qlen) return;
    const int64_t prow = ((int64_t)(q0 + qi) * nq + head) * Z + slice;
    if (hi == 0) {
      part_ml[2 * prow] = l != l ? INFINITY : m;         // a NaN is the merged row's too
      part_ml[2 * prow + 1] = l;
    }
    float* dst = part_o + prow * D + 4 * hi;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(dst + 32 * t + 8 * j) = f32x4{o[t][4 * j], o[t][4 * j + 1], o[t][4 * j + 2], o[t][4 * j + 3]};
    return;
  }
  // The rows meet in LDS, to leave it whole (stored by 8 bytes of 32 rows at a time 32 x 512 takes 113.6 us, so 103; 64 rows alone 6.7 -> 5.7).
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  static_assert(64 * KST <= KV4_BN * KST && 64 * KST <= KV4_BN * VST, "two waves' rows in each tile");
  __syncthreads();
  T* rows = (wave < 2 ? lds_k[0] : lds_v[0]) + (wave & 1) * 32 * KST;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      Pack4<T> pk;
#pragma unroll
      for (int i = 0; i < 4; ++i) pk.h[i] = from_f<T>(o[t][4 * j + i] * inv);
      *reinterpret_cast<u32x2*>(rows + col * KST + 32 * t + 8 * j + 4 * hi) = pk.u;
    }
  asm volatile("" ::: "memory");                         // the wave's own rows: its LDS operations are in order
  constexpr int LPR = D / 8, RPI = 64 / LPR;             // lanes per row, rows at a time
#pragma unroll
  for (int i = 0; i < 32 / RPI; ++i) {
    const int r = i * RPI + lane / LPR;
    const u32x4 x = *reinterpret_cast<const u32x4*>(rows + r * KST + lane % LPR * 8);
    if (wrow + r < qlen)
      *reinterpret_cast<u32x4*>(out + ((int64_t)(q0 + wrow + r) * nq + head) * D + lane % LPR * 8) = x;
  }
}

// D / 4 threads per row of a work item's block and head, four elements each; slices' partials eight at a time.
template <typename T, int D>
__global__ __launch_bounds__(256) void kv4_prefill_merge_kernel(
    T* __restrict__ out, const float* __restrict__ part_o, const float* __restrict__ part_ml, const int* __restrict__ qsl,
    const int* __restrict__ seq_lens, const int* __restrict__ work_seq, const int* __restrict__ work_mblk, int nq, int cap,
    int seqs, int rows_all, int Z) {
  constexpr int ROWS = 256 / (D / 4), ZB = 8;
  const int item = blockIdx.x / nq, head = blockIdx.x % nq;
  const int seq = work_seq[item], mb = work_mblk[item];
  if (seq < 0 || seq >= seqs || mb < 0) return;
  const int q0 = qsl[seq], q1 = qsl[seq + 1];
  if (q0 < 0 || q1 <= q0 || q1 > rows_all || min(seq_lens[seq], cap) < q1 - q0 || mb > (q1 - q0 - 1) / KV4_BM) return;
  const int r = mb * KV4_BM + blockIdx.y * ROWS + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
  if (r >= q1 - q0) return;                              // as the kernel above
  const int64_t row = ((int64_t)(q0 + r) * nq + head) * Z;
  float top = -INFINITY, total = 0.f;
  for (int z = 0; z < Z; ++z) top = fmaxf(top, part_ml[2 * (row + z)]);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int z0 = 0; z0 < Z; z0 += ZB) {
    float m[ZB], l[ZB];
    f32x4 v[ZB];
#pragma unroll
    for (int i = 0; i < ZB; ++i) {
      const int z = min(z0 + i, Z - 1);
      m[i] = part_ml[2 * (row + z)];
      l[i] = part_ml[2 * (row + z) + 1];
      v[i] = *reinterpret_cast<const f32x4*>(part_o + (row + z) * D + d);
    }
#pragma unroll
    for (int i = 0; i < ZB; ++i) {
      // a slice that saw nothing has zeros; one that saw a NaN has m = inf, and its row is NaN
      const float f = z0 + i < Z && m[i] != -INFINITY ? __builtin_amdgcn_exp2f(m[i] - top) : 0.f;
      total += f * l[i];
      acc += v[i] * f;
    }
  }
  const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
  Pack4<T> pk;
#pragma unroll
  for (int i = 0; i < 4; ++i) pk.h[i] = from_f<T>(acc[i] * inv);
  *reinterpret_cast<u32x2*>(out + row / Z * D + d) = pk.u;
}

template <typename T, int D>
static void kv4_prefill_dispatch(const Kv4Prefill& a, float sl2, hipStream_t s) {
  const int G = a.nq / a.nkv;
  // One buffer per tile: three workgroups of heads of 128 fit a CU (four of 64), which fill each other's waits; two, and a barrier less
  // per tile, where there are not more workgroups than two per CU: two buffers -> one, us: 4 x 4096 543 -> 522, 32 x 512 121.5 ->
  // 113; 64 rows alone 6.2 -> 6.9, 512 18.0 -> 19.5, 2048 55 -> 61.
#define KGC_KV4_PF_B(GH, BUFS)                                                                                        \
  kv4_prefill_kernel<T, D, GH, BUFS><<<blocks, 256, 0, s>>>(                                                            \
      (const T*)a.q, (T*)a.out, (const uint8_t*)a.k_cache, (const uint8_t*)a.v_cache, a.block_tables, a.bt_stride,      \
      a.query_start_loc, a.seq_lens, a.work_seq, a.work_mblk, a.nq, a.nkv, a.bs_log2, sl2, a.num_blocks, a.seqs,        \
      a.rows, a.part_o, a.part_ml, a.Z)
#define KGC_KV4_PF(GH)                                                                                                \
  const int blocks = a.n_work * (a.nkv * (G / GH) * GH * a.Z);                                                          \
  if (blocks <= 2 * device_cus()) KGC_KV4_PF_B(GH, 2);                                                                  \
  else KGC_KV4_PF_B(GH, 1)
  if (G % 4 == 0) {
    KGC_KV4_PF(4);
  } else if (G % 2 == 0) {
    KGC_KV4_PF(2);
  } else {
    KGC_KV4_PF(1);
  }
#undef KGC_KV4_PF_B
#undef KGC_KV4_PF
  if (a.Z > 1)
    kv4_prefill_merge_kernel<T, D><<<dim3(a.n_work * a.nq, KV4_BM / (1024 / D)), 256, 0, s>>>(
        (T*)a.out, a.part_o, a.part_ml, a.query_start_loc, a.seq_lens, a.work_seq, a.work_mblk, a.nq,
        a.bt_stride << a.bs_log2, a.seqs, a.rows, a.Z);
}

void launch_kv4_prefill(int dtype, const Kv4Prefill& a, float scale, hipStream_t s) {
  if (a.n_work == 0) return;
  const float sl2 = scale * 1.4426950408889634f;
  if (dtype == DT_BF16) {
    if (a.D == 128) kv4_prefill_dispatch<bf16, 128>(a, sl2, s);
    else kv4_prefill_dispatch<bf16, 64>(a, sl2, s);
  } else {
    if (a.D == 128) kv4_prefill_dispatch<f16, 128>(a, sl2, s);
    else kv4_prefill_dispatch<f16, 64>(a, sl2, s);
  }
}

KGC_DEBUG_TU(kv4_prefill)

}  // namespace kgc
