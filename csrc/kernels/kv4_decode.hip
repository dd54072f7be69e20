// Paged-attention decode over the 4-bit cache (kv4.h): one query row per sequence.
//
// A workgroup of NW waves per (sequence, kv head, z-slice), with the slices and the merge of paged_decode_wave_kernel
// (decode_slices.h, attention_decode.hip); its waves share the slice's chunks and merge in LDS, so that most calls are one
// launch.  A chunk is 32 tokens, two groups of 16; a page holds 16 or more, so that a group lies in one.  Lane (token r16 of a
// group, quarter qd of the head) loads its quarter row with one load of D / 8 bytes, and the scale with it; next chunk's loads are
// on their way while one computes.
//   S^T[token][head] = K Q^T: the quarter row, widened, is the operand of D / 32 MFMAs as it is -- their contraction takes the
//                      head's elements in the order (quarter, 8 of it, next 8 ..), and so does q's operand
//   O^T[d][head]    += V^T P^T: the widened rows go through LDS, where the transposing reads make columns of them; the
//                      contraction's order of tokens is that of S^T's accumulator, so that P needs no exchange
#include "common.h"
#include "decode_slices.h"
#include "kv4.h"
#include "launch.h"

namespace kgc {

__device__ __forceinline__ float kv4_max_rows(float x) {     // over the four lanes that share lane & 15
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW, 2) void kv4_decode_kernel(
    T* __restrict__ out, const T* __restrict__ q, const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
    const int* __restrict__ block_tables, int bt_stride, const int* __restrict__ ctx_lens, float* __restrict__ max_logits,
    float* __restrict__ exp_sums, float* __restrict__ tmp_out, int nq, int nkv, int bs_log2, float scale_log2,
    int num_blocks, DecodeLeast least) {
  typedef typename Vec8<T>::type V8;
  constexpr int KS = D / 32, DT = D / 16, VS = D + 16;       // VS: the 4 rows x 32 bytes of a transposing read on 32 banks
  constexpr int OS = D + 4;                                  // floats of a head's row where the waves meet
  static_assert(32 * VS * sizeof(T) >= 16 * OS * sizeof(float), "a wave's results in its own V rows");
  __shared__ __attribute__((aligned(16))) T all_v[NW][32 * VS];
  __shared__ float all_m[NW][16], all_l[NW][16];
  const int b = blockIdx.x, h = blockIdx.y, z = blockIdx.z, Z = gridDim.z;
  const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r16 = lane & 15, qd = lane >> 4;
  T* lds_v = all_v[wave];
  const int G = nq / nkv;
  int ctx_in = ctx_lens[b];
  KGC_DCHECK_RANGE(ctx_in, 0, (bt_stride << bs_log2) + 1, "decode ctx_len");
  const int ctx = min(ctx_in, bt_stride << bs_log2);         // a bad length gives wrong output, never a fault
  const int* bt = block_tables + (int64_t)b * bt_stride;
  const int bs = 1 << bs_log2, bsm = bs - 1;
  const int64_t page_bytes = kv4_page_bytes(bs, D);

  const int nchunk = (max(ctx, 0) + 31) >> 5;
  const int min_per = decode_min_chunks(least, nchunk);
  const int per = decode_slice_chunks(nchunk, Z, min_per);
  const int nused = decode_used_slices(nchunk, Z, min_per);
  const int s0 = min(nchunk, z * per), s1 = min(nchunk, s0 + per);
  if (s0 >= s1 && (z > 0 || nchunk > 0)) return;             // the whole workgroup: an empty slice is not merged
  const int c0 = s0 + (s1 - s0) * wave / NW, c1 = s0 + (s1 - s0) * (wave + 1) / NW;
  const int end = min(ctx, c1 << 5);                         // this wave's tokens: [32 c0, end)

  struct Frag {
    uint32_t k[2][KS], v[2][KS];
    uint8_t ks[2], vs[2];
  };
  auto load = [&](uint32_t (&w)[KS], const uint8_t* p) {
    if constexpr (KS == 4) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(p);
      w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    } else {
      const u32x2 x = *reinterpret_cast<const u32x2*>(p);
      w[0] = x.x; w[1] = x.y;
    }
  };
  auto issue = [&](Frag& f, int ci) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      // tokens behind the slice's last one are that one again: their scores are masked
      const int t0 = min((ci << 5) + 16 * g, end - 1), tok = min((ci << 5) + 16 * g + r16, end - 1);
      const int64_t page = ((int64_t)kv4_page(bt, t0 >> bs_log2, bt_stride, num_blocks) * nkv + h) * page_bytes;
      const int row = tok & bsm;
      const int at = row * (D / 2) + qd * (D / 8), sc = bs * (D / 2) + row * (D / 32) + (qd * D / 4) / 32;
      load(f.k[g], kc + page + at);
      load(f.v[g], vc + page + at);
      f.ks[g] = kc[page + sc];
      f.vs[g] = vc[page + sc];
    }
  };

  float m_run = -INFINITY, l_run = 0.f;
  f32x4 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  Pack8<T> qf[KS];
  const T* qrow = q + ((int64_t)b * nq + h * G + (r16 < G ? r16 : 0)) * D + qd * (D / 4);
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s].u = *reinterpret_cast<const u32x4*>(qrow + 8 * s);
  Frag fa, fb;
  if (c0 < c1) {
    issue(fa, c0);
    issue(fb, min(c0 + 1, c1 - 1));
  }
  // q is there before the loop: a wait for it in there would be one for the newest chunk's loads, too
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    asm volatile("" : "+v"(qf[s].u));
    if (r16 >= G) qf[s].u = u32x4{0, 0, 0, 0};
  }
  auto compute = [&](const Frag& f, int ci) {
    const int base = ci << 5;
    f32x4 sc[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const float size = kv4_scale(f.ks[g]);
      sc[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        Pack8<T> kf;
        kf.u = fp4x8_widen<T>(f.k[g][s], size);
        sc[g] = mfma16x16x32(kf.v, qf[s].v, sc[g]);
      }
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const float size = kv4_scale(f.vs[g]);
#pragma unroll
      for (int s = 0; s < KS; ++s)
        *reinterpret_cast<u32x4*>(lds_v + (16 * g + r16) * VS + qd * (D / 4) + 8 * s) = fp4x8_widen<T>(f.v[g][s], size);
    }
    asm volatile("" ::: "memory");          // one wave: its LDS operations are in order
    float m = m_run;
    if (base + 32 <= end) {
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[g][i] *= scale_log2;
          m = fmaxf(m, sc[g][i]);
        }
    } else {
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[g][i] = base + 16 * g + 4 * qd + i < end ? sc[g][i] * scale_log2 : -INFINITY;
          m = fmaxf(m, sc[g][i]);
        }
    }
    m = kv4_max_rows(m);
    // The reference moves only where the maximum is more than 2^8 above it: probabilities are then at most 2^8, and O is seldom
    // rescaled.
    if (__any(m > m_run + 8.f)) {
      const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m);
      m_run = m;
      l_run *= f;
#pragma unroll
      for (int t = 0; t < DT; ++t) o[t] *= f;
    }
    // a row none of whose scores is above -inf (q or k too large): no difference of infinities
    const float ref = m_run == -INFINITY ? 0.f : m_run;
    // probabilities are rounded to T for the product, as the keys' and values' type has it; the sum, in 32 bits, is that of the
    // rounded ones, so that they add up to one
    Pack8<T> pf;
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) pf.h[4 * g + i] = from_f<T>(__builtin_amdgcn_exp2f(sc[g][i] - ref));
#pragma unroll
    for (int i = 0; i < 4; ++i) l_run = kv4_add_pair<T>(pf.u[i], l_run);
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const T* src = lds_v + (4 * qd + (r16 >> 2)) * VS + 16 * t + 4 * (r16 & 3);
      const u32x2 lo = ld_tr4(src), hi = ld_tr4(src + 16 * VS);
      Pack8<T> vf;
      vf.u = u32x4{lo.x, lo.y, hi.x, hi.y};
      o[t] = mfma16x16x32(vf.v, pf.v, o[t]);
    }
    asm volatile("" ::: "memory");
  };
  // straight-line, two chunks deep: behind the last one a chunk is computed masked (p = 0, alpha = 1)
  for (int ci = c0; ci < c1; ci += 2) {
    compute(fa, ci);
    issue(fa, min(ci + 2, c1 - 1));
    compute(fb, ci + 1);
    issue(fb, min(ci + 3, c1 - 1));
  }

  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  const bool whole = Z == 1 || nused == 1;  // the merge skips such a row
  if constexpr (NW > 1) {
    float* mine = reinterpret_cast<float*>(lds_v);
#pragma unroll
    for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4*>(mine + r16 * OS + 16 * t + 4 * qd) = o[t];
    if (qd == 0) {
      all_m[wave][r16] = m_run;
      all_l[wave][r16] = l_run;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < G * (D / 4); e += 64 * NW) {
      const int g = e / (D / 4), d = e % (D / 4) * 4;
      float top = all_m[0][g];
#pragma unroll
      for (int w = 1; w < NW; ++w) top = fmaxf(top, all_m[w][g]);
      const float ref = top == -INFINITY ? 0.f : top;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = __builtin_amdgcn_exp2f(all_m[w][g] - ref);
        acc += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(all_v[w]) + g * OS + d) * f;
        sum += all_l[w][g] * f;
      }
      const int64_t row = (int64_t)b * nq + h * G + g;
      if (whole) {
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        Pack4<T> pk;
#pragma unroll
        for (int i = 0; i < 4; ++i) pk.h[i] = from_f<T>(acc[i] * inv);
        *reinterpret_cast<u32x2*>(out + row * D + d) = pk.u;
      } else {
        const int64_t prow = row * Z + z;
        *reinterpret_cast<f32x4*>(tmp_out + prow * D + d) = acc;
        if (d == 0) {
          max_logits[prow] = sum != sum ? INFINITY : top;    // a NaN is the merged row's too
          exp_sums[prow] = sum;
        }
      }
    }
    return;
  }
  const int64_t row = (int64_t)b * nq + h * G + r16;
  if (whole) {
    if (z > 0 || r16 >= G) return;
    const float inv = l_run > 0.f || l_run != l_run ? 1.f / l_run : 0.f;
    T* orow = out + row * D + 4 * qd;
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      Pack4<T> pk;
#pragma unroll
      for (int i = 0; i < 4; ++i) pk.h[i] = from_f<T>(o[t][i] * inv);
      *reinterpret_cast<u32x2*>(orow + 16 * t) = pk.u;
    }
    return;
  }
  if (z >= nused || r16 >= G) return;
  const int64_t prow = row * Z + z;
  float* dst = tmp_out + prow * D + 4 * qd;
#pragma unroll
  for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4*>(dst + 16 * t) = o[t];
  if (qd == 0) {
    max_logits[prow] = l_run != l_run ? INFINITY : m_run;
    exp_sums[prow] = l_run;
  }
}

template <typename T, int D>
static void kv4_decode_dispatch(const Kv4Decode& a, int waves, DecodeLeast least, float sl2, hipStream_t s) {
#define KGC_KV4_DEC(NW)                                                                                                \
  kv4_decode_kernel<T, D, NW><<<dim3(a.B, a.nkv, a.Z), 64 * NW, 0, s>>>(                                                         \
      (T*)a.out, (const T*)a.q, (const uint8_t*)a.k_cache, (const uint8_t*)a.v_cache, a.block_tables, a.bt_stride,      \
      a.ctx_lens, a.max_logits, a.exp_sums, a.tmp_out, a.nq, a.nkv, a.bs_log2, sl2, a.num_blocks, least)
  if (waves == 8) KGC_KV4_DEC(8);
  else if (waves == 4) KGC_KV4_DEC(4);
  else if (waves == 2) KGC_KV4_DEC(2);
  else KGC_KV4_DEC(1);
#undef KGC_KV4_DEC
}

// Waves per workgroup (ops/__init__.py has the same numbers, and chooses Z by them).  us, 8 kv heads of 128 unless said, one
// launch or, with ->, two:
//   fewer than 64 pairs leave CUs free for slices, and four waves meet sooner than eight: 1 x 128 4.9 (eight 5.9), 1 x 2000 eight slices
//     -> 7.6 (9.2), 4 x 1000 -> 8.3 (9.7);
//   up to 512 eight waves take the place of slices: 32 x 2000 16.7 (four 18.2, four and two slices -> 21.8), 33 x 1001 of 12 heads of
//     64 10.4 (10.5, -> 12.2);
//   from 512 on the LDS of eight (two workgroups per CU) makes short contexts wait: 64 x 512 10.5 (11.1), 64 x 8192 96.2 (97.0);
//   from 1024 on two: 128 x 1000 27.2 (one 29.2, four 27.7), 160 x 1000 33.4 (35.7, 36.4), 128 x 4000 93.1 (99.4, 95.6), 100 x 1000 of
//     12 heads of 64 22.3 (26.5, 22.9), 128 x 300 12.6 (12.5, 13.6); a short context pays for it, 128 x 60 7.5 (6.1, 7.8);
//   from 1536 on a wave has a pair to itself: 256 x 60 7.9 (two 10.6, four 13.6), 256 x 640 33.5 (34.8, 38.6), 200 x 1000 42.3
//     (43.1, 43.2), 250 x 500 of 12 heads of 64 25.6 (27.3, 30.7), 130 x 1000 of them 28.3 (28.3, 29.7).
static int kv4_decode_waves(int64_t pairs) { return pairs >= 1536 ? 1 : pairs >= 1024 ? 2 : pairs >= 512 ? 4 : pairs >= 64 ? 8 : 4; }

void launch_kv4_decode(int dtype, const Kv4Decode& a, float scale, hipStream_t s) {
  if (a.B == 0) return;
  const int64_t pairs = (int64_t)a.B * a.nkv;
  const int waves = kv4_decode_waves(pairs);
  // Slices hold two chunks (the pipeline) for each wave or more, and contexts of up to 16 chunks, 64 from 64 pairs on, are one:
  // 1 x 500 6.3 us whole, 7.5 as two with their merge; 16 x 2000 13.5 and 13.4.
  const DecodeLeast least{pairs >= 64 ? 64 : 16, 2 * waves, 2 * waves};
  const float sl2 = scale * 1.4426950408889634f;
  if (dtype == DT_BF16) {
    if (a.D == 128) kv4_decode_dispatch<bf16, 128>(a, waves, least, sl2, s);
    else kv4_decode_dispatch<bf16, 64>(a, waves, least, sl2, s);
  } else {
    if (a.D == 128) kv4_decode_dispatch<f16, 128>(a, waves, least, sl2, s);
    else kv4_decode_dispatch<f16, 64>(a, waves, least, sl2, s);
  }
  if (a.Z > 1)
    launch_paged_decode_merge(dtype, a.out, a.max_logits, a.exp_sums, a.tmp_out, a.ctx_lens, a.B, a.nq, a.D, a.Z,
                              a.bt_stride << a.bs_log2, least, s);
}

KGC_DEBUG_TU(kv4_decode)

}  // namespace kgc
