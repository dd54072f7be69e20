// Writing and reading the 4-bit key / value cache (kv4.h).
//
// kv4_write_kernel: q, k, v of a step from the rows of its fused QKV projection, as rope_kv_kernel (rope_cache.hip) for the
// wider caches: optional per-head RMS norm, NeoX rotation by one position or by one per axis, q stored in T, k and v as
// e2m1 numbers with their scales.  A thread has the 16-byte chunk pair (c, c + d / 2) of HG heads that lie side by side in the
// row: the pair is what the rotation needs, four neighbouring lanes hold a block of 32, and cos / sin are loaded once
// for the heads.  A wave has the same heads of 8 tokens (16 with heads of 64), so that its lanes take the same way and a page's
// rows are written side by side.
//
// k is rotated in 64 bits, where the products are exact, and their sum is rounded to odd: the nearest code of that is the nearest code of
// the exact sum, also where a key lies next to the border of two codes (which are up to a third apart) by less than 64 bits
// hold, and whatever order of operations a compiler prefers.  (Rounding the sum to 64 bits first takes 95.8 us where this takes 98.5, 16384
// rows with their reads; one branch for a thread's 16 sums instead of one each keeps more registers: 101.8.)  Values, and keys that are
// not rotated, are numbers of T already.
#include "common.h"
#include "kv4.h"
#include "launch.h"
#include "rope_axes.h"

namespace kgc {

constexpr int KV4_NT = 256;

// RS: rows are times row_scale[t] before they are rounded to T (a template: a branch in here costs 2000 rows 20.3 -> 22.1 us).
template <typename T, bool NORM, bool ROPE, bool SL, bool AXES, int HG, bool RS>
__global__ __launch_bounds__(KV4_NT) void kv4_write_kernel(
    const void* __restrict__ qkv, int64_t qkv_stride, int S, int64_t slice_stride, const int64_t* __restrict__ positions,
    const float* __restrict__ cos_sin, T* __restrict__ q_out, uint8_t* __restrict__ k_cache, uint8_t* __restrict__ v_cache,
    const int64_t* __restrict__ slot_mapping, const T* __restrict__ qn_w, const T* __restrict__ kn_w,
    const float* __restrict__ row_scale, int64_t T_, int nq, int nkv, int d, int bs, float eps, int num_blocks, RopeAxes ax) {
  const int tph = d >> 4, half = d >> 1;               // threads per head: 4 or 8, whole lane groups
  const int heads = nq + 2 * nkv, groups = (heads + HG - 1) / HG, tpw = 64 / tph;
  const int64_t wave = (int64_t)blockIdx.x * (KV4_NT / 64) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, c = lane % tph;
  const int64_t t = wave / groups * tpw + lane / tph;
  if (t >= T_) return;                                 // whole lane groups
  const int h0 = (int)(wave % groups) * HG;
  const int64_t row = t * qkv_stride;
  int64_t slot = slot_mapping[t];
  if (slot >= (int64_t)num_blocks * bs) slot = -1;     // beyond the pool: not written
  const int64_t blk = slot >= 0 ? slot / bs : 0;
  const int off = slot >= 0 ? (int)(slot - blk * bs) : 0;
  float by = 1.f;
  if constexpr (RS) by = row_scale[t];
  auto load8 = [&](int col) -> u32x4 {
    if constexpr (!SL) {
      Pack8<T> o;
      o.u = *reinterpret_cast<const u32x4*>(reinterpret_cast<const T*>(qkv) + row + col);
      if constexpr (RS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) o.h[j] = from_f<T>(to_f(o.h[j]) * by);
      }
      return o.u;
    } else {
      const float* p = reinterpret_cast<const float*>(qkv) + row + col;
      f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
      for (int z = 1; z < S; ++z) {
        a += *reinterpret_cast<const f32x4*>(p + z * slice_stride);
        b += *reinterpret_cast<const f32x4*>(p + z * slice_stride + 4);
      }
      if constexpr (RS) {
        a *= by;
        b *= by;
      }
      Pack8<T> o;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        o.h[q] = from_f<T>(a[q]);
        o.h[4 + q] = from_f<T>(b[q]);
      }
      return o.u;
    }
  };
  Pack8<T> a[HG], b[HG];
#pragma unroll
  for (int k = 0; k < HG; ++k) {                       // the last group's missing heads: its last one again
    const int col = min(h0 + k, heads - 1) * d + c * 8;
    a[k].u = load8(col);
    b[k].u = load8(col + half);
  }
  float cc[8], sn[8];
  if constexpr (ROPE) {
    if (h0 < nq + nkv) {
      if constexpr (AXES) {
        axes_cos_sin(ax, positions, (int)t, cos_sin, d, c * 8, cc, sn);
      } else {
        int64_t p = positions[t];
        KGC_DCHECK_RANGE(p, 0, ax.rows, "position");
        const float* cs = cos_sin + min(max(p, (int64_t)0), (int64_t)ax.rows - 1) * d + c * 8;
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(cs + j), y = *reinterpret_cast<const f32x4*>(cs + half + j);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            cc[j + i] = x[i];
            sn[j + i] = y[i];
          }
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < HG; ++k) {
    const int head = h0 + k;                           // the same for the head's lanes
    if (head >= heads) break;
    float xa[8], xb[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      xa[j] = to_f(a[k].h[j]);
      xb[j] = to_f(b[k].h[j]);
    }
    if (NORM && head < nq + nkv) {
      const T* w = head < nq ? qn_w : kn_w;
      Pack8<T> wa, wb;
      wa.u = *reinterpret_cast<const u32x4*>(w + c * 8);
      wb.u = *reinterpret_cast<const u32x4*>(w + half + c * 8);
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += xa[j] * xa[j] + xb[j] * xb[j];
      for (int o = 1; o < tph; o <<= 1) ss += __shfl_xor(ss, o, 64);
      const float inv = rsqrtf(ss / (float)d + eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) {                    // the norm's own result is one of T
        xa[j] = to_f(from_f<T>(xa[j] * inv * to_f(wa.h[j])));
        xb[j] = to_f(from_f<T>(xb[j] * inv * to_f(wb.h[j])));
      }
    }
    if (head < nq) {
      if constexpr (ROPE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) neox_rot(xa[j], xb[j], cc[j], sn[j], xa[j], xb[j]);
      }
      Pack8<T> oa, ob;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        oa.h[j] = from_f<T>(xa[j]);
        ob.h[j] = from_f<T>(xb[j]);
      }
      T* dst = q_out + (t * nq + head) * d + c * 8;
      *reinterpret_cast<u32x4*>(dst) = oa.u;
      *reinterpret_cast<u32x4*>(dst + half) = ob.u;
      continue;
    }
    const bool key = head < nq + nkv;
    if constexpr (ROPE) {
      if (key) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const double x = xa[j], y = xb[j], co = cc[j], si = sn[j];
          xa[j] = sum_to_odd(x * co, -(y * si));
          xb[j] = sum_to_odd(y * co, x * si);
        }
      }
    }
    float ma = 0.f, mb = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {                      // e2m1 has no NaN: zero
      xa[j] = xa[j] == xa[j] ? xa[j] : 0.f;
      xb[j] = xb[j] == xb[j] ? xb[j] : 0.f;
      ma = fmaxf(ma, fabsf(xa[j]));
      mb = fmaxf(mb, fabsf(xb[j]));
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      ma = fmaxf(ma, __shfl_xor(ma, o, 64));
      mb = fmaxf(mb, __shfl_xor(mb, o, 64));
    }
    if (slot < 0) continue;
    const uint32_t sa = kv4_scale_byte<T>(ma), sb = kv4_scale_byte<T>(mb);
    uint8_t* page = (key ? k_cache : v_cache) + (blk * nkv + (key ? head - nq : head - nq - nkv)) * kv4_page_bytes(bs, d);
    uint32_t* dst = reinterpret_cast<uint32_t*>(page + off * (d >> 1));
    dst[c] = fp4x8(xa, kv4_scale(sa));
    dst[tph + c] = fp4x8(xb, kv4_scale(sb));
    if ((c & 3) == 0) {
      uint8_t* sc = page + bs * (d >> 1) + off * (d >> 5);
      sc[c >> 2] = (uint8_t)sa;
      sc[(tph + c) >> 2] = (uint8_t)sb;
    }
  }
}

// Rows of the cache as the values they stand for; slots outside the pool give zeros.  8 elements a thread, U times.
template <typename T, int U>
__global__ __launch_bounds__(KV4_NT) void kv4_read_kernel(T* __restrict__ out, const uint8_t* __restrict__ cache,
                                                          const int64_t* __restrict__ slots, int64_t n, int nkv, int d,
                                                          int bs, int num_blocks) {
  const int per = nkv * (d >> 3);
  const int64_t first = (int64_t)blockIdx.x * (KV4_NT * U) + threadIdx.x;
  int64_t at[U];
  int off[U], c[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = min(first + u * KV4_NT, n * per - 1) / per;
    at[u] = slots[i];
  }
  uint32_t w[U];
  uint8_t s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t item = min(first + u * KV4_NT, n * per - 1);
    const int r = (int)(item % per), h = r / (d >> 3);
    c[u] = r % (d >> 3);
    const bool there = at[u] >= 0 && at[u] < (int64_t)num_blocks * bs;
    if (!there) at[u] = 0;                             // (a pool without pages has no slots: nothing is launched)
    const int64_t blk = at[u] / bs;
    off[u] = (int)(at[u] - blk * bs);
    const uint8_t* page = cache + (blk * nkv + h) * kv4_page_bytes(bs, d);
    w[u] = reinterpret_cast<const uint32_t*>(page + off[u] * (d >> 1))[c[u]];
    s[u] = page[bs * (d >> 1) + off[u] * (d >> 5) + (c[u] >> 2)];
    if (!there) w[u] = 0, s[u] = 127;
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (first + u * KV4_NT < n * per) reinterpret_cast<u32x4*>(out)[first + u * KV4_NT] = fp4x8_widen<T>(w[u], kv4_scale(s[u]));
}

template <typename T, bool SL, bool AXES, int HG, bool RS = false>
static void kv4_write_norm(const Kv4Write& w, const RopeAxes& ax, int64_t blocks, hipStream_t s) {
#define KGC_KV4_WRITE(N, R)                                                                                            \
  kv4_write_kernel<T, N, R, SL, AXES, HG, RS><<<(unsigned)blocks, KV4_NT, 0, s>>>(                                          \
      w.qkv, w.qkv_stride, w.S, w.slice_stride, w.positions, w.cos_sin, (T*)w.q_out, (uint8_t*)w.k_cache,               \
      (uint8_t*)w.v_cache, w.slots, (const T*)w.q_norm_w, (const T*)w.k_norm_w, w.row_scale, w.T, w.nq, w.nkv, w.d,     \
      w.bs, w.eps, w.num_blocks, ax)
  if constexpr (AXES) {
    if (w.q_norm_w) KGC_KV4_WRITE(true, true);
    else KGC_KV4_WRITE(false, true);
  } else if (w.q_norm_w) {
    if (w.use_rope) KGC_KV4_WRITE(true, true);
    else KGC_KV4_WRITE(true, false);
  } else {
    if (w.use_rope) KGC_KV4_WRITE(false, true);
    else KGC_KV4_WRITE(false, false);
  }
#undef KGC_KV4_WRITE
}

template <typename T>
static void kv4_write_dispatch(const Kv4Write& w, const RopeAxes& ax, hipStream_t s) {
  const int64_t tokens = (w.T * (w.d >> 4) + 63) / 64;           // in waves' worth
  auto blocks = [&](int hg) { return (tokens * ((w.nq + 2 * w.nkv + hg - 1) / hg) + KV4_NT / 64 - 1) / (KV4_NT / 64); };
  if (w.row_scale) {                                             // (the host: no sections)
    if (w.S > 0) kv4_write_norm<T, true, false, 1, true>(w, ax, blocks(1), s);
    else kv4_write_norm<T, false, false, 1, true>(w, ax, blocks(1), s);
  } else if (w.S > 0) {
    if (ax.n) kv4_write_norm<T, true, true, 1>(w, ax, blocks(1), s);
    else kv4_write_norm<T, true, false, 1>(w, ax, blocks(1), s);
  } else if (blocks(1) <= 4096) {
    // Few workgroups: a head per thread, all loads of a call on their way at once; many: cos / sin for four.  us with both
    // caches' rows read back, one head -> four: 256 rows of 32 / 8 heads 9.2 -> 12.7, 1000 13.4 -> 16.2, 2000 20.2 -> 20.2, 2700 26.3
    // -> 25.9, 4000 33.9 -> 34.2, 16384 107 -> 98.0 (the write alone 77, 353 MB); 4000 of 12 / 12 heads of 64 19.7 -> 23.3.
    if (ax.n) kv4_write_norm<T, false, true, 1>(w, ax, blocks(1), s);
    else kv4_write_norm<T, false, false, 1>(w, ax, blocks(1), s);
  } else if (ax.n) {
    kv4_write_norm<T, false, true, 4>(w, ax, blocks(4), s);
  } else {
    kv4_write_norm<T, false, false, 4>(w, ax, blocks(4), s);
  }
}

void launch_kv4_write(int dtype, const Kv4Write& w, const RopeAxes& ax, hipStream_t s) {
  if (w.T == 0) return;
  if (dtype == DT_BF16) kv4_write_dispatch<bf16>(w, ax, s);
  else kv4_write_dispatch<f16>(w, ax, s);
}

template <typename T>
static void kv4_read_dispatch(void* out, const void* cache, const int64_t* slots, int64_t n, int nkv, int d, int bs,
                              int num_blocks, hipStream_t s) {
  const int64_t items = n * nkv * (d >> 3);
  if (items < (1 << 20))
    kv4_read_kernel<T, 1><<<(unsigned)((items + KV4_NT - 1) / KV4_NT), KV4_NT, 0, s>>>(
        (T*)out, (const uint8_t*)cache, slots, n, nkv, d, bs, num_blocks);
  else
    kv4_read_kernel<T, 4><<<(unsigned)((items + 4 * KV4_NT - 1) / (4 * KV4_NT)), KV4_NT, 0, s>>>(
        (T*)out, (const uint8_t*)cache, slots, n, nkv, d, bs, num_blocks);
}

void launch_kv4_read(int dtype, void* out, const void* cache, const int64_t* slots, int64_t n, int nkv, int d, int bs,
                     int num_blocks, hipStream_t s) {
  if (n == 0 || num_blocks == 0) return;
  if (dtype == DT_BF16) kv4_read_dispatch<bf16>(out, cache, slots, n, nkv, d, bs, num_blocks, s);
  else kv4_read_dispatch<f16>(out, cache, slots, n, nkv, d, bs, num_blocks, s);
}

KGC_DEBUG_TU(kv4_cache)

}  // namespace kgc
