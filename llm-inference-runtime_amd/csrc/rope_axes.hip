// RoPE whose frequencies turn by positions of several axes (time, height and
// width of a token of an image or a video), in place on q and k, alone or with
// the page append of the k and v rows.
//
// Frequency i of a token t turns by axis_pos[a(i)][t] / rope_scale *
// theta^(-2 i / rotary_dim).  a(i): the axes take blocks of `share[a]`
// frequencies one after the other or, cyclic, axis i mod n takes frequency i
// while i < n share[axis], and axis 0 the others.  Elements past rotary_dim are
// left as they are.
//
// Bound by HBM for prompts (each row read once, q and k rows written once, k and
// v rows written to their pages: 21 181 tokens of 32/8 heads, D = 128, 564 MB in
// 100 us, 5.6 TB/s, where a large copy moves 4.8) and by one load-to-store chain
// for a decode step's rows (33 of 32/4 heads, D = 64: 4.4 us).  The work is split as in the RoPE + append of one position
// (misc.hip): a workgroup owns T tokens (launch_rope_axes); 8 lanes (fewer where a head has fewer
// chunk pairs) work a head, each with two 16-byte chunks; the cosines and sines
// are evaluated once per (token, frequency), one per lane, into LDS while the first
// rows are on their way.
#include <algorithm>
#include <cmath>

#include "append.h"

namespace pa {

constexpr int kMaxAxes = 4;
constexpr int kAxesFreqs = 64;   // frequencies of a workgroup (8 chunk pairs)
constexpr int kAxesBatch = 4;    // heads a thread has in flight
constexpr int kAxesTokens = 16;  // tokens of a workgroup at most
constexpr int kAxesThreads = 256;
constexpr int kAxesSpread = 512;   // workgroups before a token shares one
constexpr int kAxesGroups = 1024;  // workgroups left by more than 4 tokens each
constexpr int kAxesFewLanes = 96;  // of a token

struct RopeAxesArgs {
  AppendArgs a;  // cache null: q and k only
  uint16_t* q;
  int64_t q_sn, q_sh;
  int32_t hq;
  const int32_t* axis_pos;  // [n_axes, nnz], rows `axis_stride` apart
  int64_t axis_stride;
  int32_t n_axes, cyclic;
  int32_t share[kMaxAxes];  // frequencies of each axis
  int32_t rotary_dim;
  int32_t tokens;   // T
  int32_t c_shift;  // log2 of the lanes per head
  double inv_scale, log2_theta;
};

__device__ __forceinline__ int axis_of(const RopeAxesArgs& r, int f) {
  if (r.cyclic) {
    const int a = f % r.n_axes;
    int share = r.share[0];
#pragma unroll
    for (int i = 1; i < kMaxAxes; ++i) share = a == i ? r.share[i] : share;
    return f < r.n_axes * share ? a : 0;
  }
  int a = 0, edge = 0;
#pragma unroll
  for (int i = 0; i < kMaxAxes - 1; ++i) {
    edge += r.share[i];
    if (f >= edge && i + 1 < r.n_axes) a = i + 1;
  }
  return a;
}

// Eight 16-bit elements holding four adjacent pairs, rotated by c[0..4), s[0..4).
template <bool IS_BF16>
__device__ __forceinline__ void rope4_adjacent(u32x4& x, const float* c, const float* s) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    float y0, y1;
    rope_rotate(h2f<IS_BF16>((uint16_t)(x[w] & 0xffffu)), h2f<IS_BF16>((uint16_t)(x[w] >> 16)),
                c[w], s[w], &y0, &y1);
    x[w] = (uint32_t)f2h<IS_BF16>(y0) | ((uint32_t)f2h<IS_BF16>(y1) << 16);
  }
}

// Lane chunk pair c of a head: the chunks at element 8 c and rotary_dim / 2
// further on where c < rotary_dim / 16, else 16 elements past rotary_dim.
// Halves (INTERLEAVE false): elements i and i + rotary_dim / 2 turn by
// frequency i.  Interleaved: elements 2 i and 2 i + 1 do.
template <bool IS_BF16, bool APPEND, bool TO_FP8, bool INTERLEAVE>
__global__ void __launch_bounds__(kAxesThreads) rope_axes_kernel(RopeAxesArgs r) {
  __shared__ __attribute__((aligned(16))) float tab[kAxesTokens][2][kAxesFreqs];
  __shared__ int64_t pages[kAxesTokens];
  __shared__ int slots[kAxesTokens];
  const AppendArgs& a = r.a;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = uniform(threadIdx.x >> 6);
  const int c0 = (int)blockIdx.y * (kAxesFreqs / 8);  // first chunk pair of this workgroup
  const int turned = r.rotary_dim / 16;               // chunk pairs that turn
  const int npair = min(kAxesFreqs / 8, a.d / 16 - c0);
  const int64_t j0 = (int64_t)blockIdx.x * r.tokens;
  const int nt = (int)min<int64_t>(r.tokens, a.nnz - j0);
  const int per_tok = r.hq + (APPEND ? 2 : 1) * a.hkv;
  const int n_units = nt * per_tok;
  const int lc = threadIdx.x & ((1 << r.c_shift) - 1);
  const int step = kAxesThreads >> r.c_shift;
  const int c = c0 + lc;
  const bool turns = c < turned;
  const int e_lo = turns ? 8 * c : r.rotary_dim + 16 * (c - turned);
  const int e_hi = turns ? e_lo + r.rotary_dim / 2 : e_lo + 8;
  const bool mine = lc < npair && (APPEND || turns);

  // unit u of the workgroup: its row, and head h: q heads, then k and v heads
  auto row_of = [&](int u, int* tok, int* h) -> uint16_t* {
    const int t = u / per_tok;
    const int x = u - t * per_tok;
    const int64_t j = j0 + t;
    *tok = t;
    *h = x;
    if (x < r.hq) return r.q + j * r.q_sn + (int64_t)x * r.q_sh;
    if (x < r.hq + a.hkv)
      return const_cast<uint16_t*>(a.k) + j * a.k_sn + (int64_t)(x - r.hq) * a.k_sh;
    return const_cast<uint16_t*>(a.v) + j * a.v_sn + (int64_t)(x - r.hq - a.hkv) * a.v_sh;
  };
  u32x4 lo[kAxesBatch], hi[kAxesBatch];
  auto load = [&](int u0) {
#pragma unroll
    for (int k = 0; k < kAxesBatch; ++k) {
      const int u = u0 + k * step;
      if (u < n_units && mine) {
        int tok, h;
        const uint16_t* x = row_of(u, &tok, &h);
        lo[k] = *reinterpret_cast<const u32x4*>(x + e_lo);
        hi[k] = *reinterpret_cast<const u32x4*>(x + e_hi);
      }
    }
  };
  int u0 = threadIdx.x >> r.c_shift;
  load(u0);
  // entry `lane` of a token's table: frequency 8 c0 + lane of the halves;
  // interleaved, the low chunks' 4 c0 + lane, then the high chunks'
  int f = 8 * c0 + lane;
  bool evaluates = f < r.rotary_dim / 2;
  if constexpr (INTERLEAVE) {
    const int part = lane & (kAxesFreqs / 2 - 1);
    f = 4 * c0 + part + (lane >= kAxesFreqs / 2 ? r.rotary_dim / 4 : 0);
    evaluates = 4 * c0 + part < r.rotary_dim / 4;
  }
  for (int t = wave; t < nt && evaluates; t += kAxesThreads / kWave) {
    float cs, sn;
    const int pos = r.axis_pos[axis_of(r, f) * r.axis_stride + j0 + t];
    rope_cos_sin(pos, f, r.rotary_dim, r.inv_scale, r.log2_theta, &cs, &sn);
    tab[t][0][lane] = cs;
    tab[t][1][lane] = sn;
  }
  if constexpr (APPEND) {
    if (wave == kAxesThreads / kWave - 1 && lane < nt) {
      int slot = 0;
      const int64_t page = append_target_page(a, (int)(j0 + lane), &slot);
      pages[lane] = page;
      slots[lane] = slot;
      count_lanes(a.err, page < 0 && blockIdx.y == 0);
    }
  }
  __syncthreads();
  while (true) {
#pragma unroll
    for (int k = 0; k < kAxesBatch; ++k) {
      const int u = u0 + k * step;
      if (u >= n_units || !mine) continue;
      int tok, h;
      uint16_t* x = row_of(u, &tok, &h);
      if (h < r.hq + a.hkv && turns) {
        if constexpr (INTERLEAVE) {
          rope4_adjacent<IS_BF16>(lo[k], &tab[tok][0][4 * lc], &tab[tok][1][4 * lc]);
          rope4_adjacent<IS_BF16>(hi[k], &tab[tok][0][kAxesFreqs / 2 + 4 * lc],
                                  &tab[tok][1][kAxesFreqs / 2 + 4 * lc]);
        } else {
          float cs[8], sn[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            cs[e] = tab[tok][0][8 * lc + e];
            sn[e] = tab[tok][1][8 * lc + e];
          }
          rope8<IS_BF16>(lo[k], hi[k], cs, sn);
        }
        *reinterpret_cast<u32x4*>(x + e_lo) = lo[k];
        *reinterpret_cast<u32x4*>(x + e_hi) = hi[k];
      }
      if (!APPEND || h < r.hq) continue;
      const int64_t page = pages[tok];
      if (page < 0) continue;
      const int kind = h >= r.hq + a.hkv ? 1 : 0;
      const int kvh = h - r.hq - kind * a.hkv;
      store_chunk<IS_BF16, TO_FP8>(a, page, slots[tok], kind, kvh, e_lo, lo[k]);
      store_chunk<IS_BF16, TO_FP8>(a, page, slots[tok], kind, kvh, e_hi, hi[k]);
    }
    u0 += kAxesBatch * step;
    if (u0 >= n_units) break;
    load(u0);
  }
}

template <bool IS_BF16, bool INTERLEAVE>
static auto* pick_rope_axes(bool append, bool fp8) {
  if (!append) return rope_axes_kernel<IS_BF16, false, false, INTERLEAVE>;
  return fp8 ? rope_axes_kernel<IS_BF16, true, true, INTERLEAVE>
             : rope_axes_kernel<IS_BF16, true, false, INTERLEAVE>;
}

// Checks of the axes, positions and rotation, and their arguments.
static int axes_setup(const char* who, const int32_t* axis_pos, int64_t axis_stride,
                      int32_t n_axes, const int32_t* share, int32_t cyclic, int32_t nnz,
                      int32_t head_dim, int32_t rotary_dim, float rope_scale, float rope_theta,
                      RopeAxesArgs* r) {
  if (rotary_dim <= 0) rotary_dim = head_dim;
  if (head_dim <= 0 || (head_dim & 15) || (rotary_dim & 15) || rotary_dim > head_dim)
    return set_error(PAGEDATTN_ERR_INVALID,
                     "%s: head_dim %d and rotary_dim %d must be multiples of 16, rotary_dim at "
                     "most head_dim",
                     who, head_dim, rotary_dim);
  if (!(rope_scale > 0.f) || !(rope_theta > 0.f))
    return set_error(PAGEDATTN_ERR_INVALID, "%s: rope_scale and rope_theta must be > 0", who);
  if (n_axes < 1 || n_axes > kMaxAxes || !share)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: %d axes (1 to %d)", who, n_axes, kMaxAxes);
  int64_t sum = 0;
  for (int i = 0; i < kMaxAxes; ++i) {
    const int x = i < n_axes ? share[i] : 0;
    if (x < 0) return set_error(PAGEDATTN_ERR_INVALID, "%s: section %d is negative", who, i);
    if (cyclic && i > 0 && x > 0 && (int64_t)n_axes * (x - 1) + i >= rotary_dim / 2)
      return set_error(PAGEDATTN_ERR_INVALID,
                       "%s: cyclic section %d of %d frequencies reaches past the %d there are", who,
                       i, x, rotary_dim / 2);
    r->share[i] = x;
    sum += x;
  }
  if (sum != rotary_dim / 2)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: sections of %lld frequencies, rotary_dim %d has %d",
                     who, (long long)sum, rotary_dim, rotary_dim / 2);
  if (nnz > 0 && !axis_pos)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: null axis positions", who);
  if (axis_stride < nnz)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: axis stride %lld below %d tokens", who,
                     (long long)axis_stride, nnz);
  r->axis_pos = axis_pos;
  r->axis_stride = axis_stride;
  r->n_axes = n_axes;
  r->cyclic = cyclic ? 1 : 0;
  r->rotary_dim = rotary_dim;
  r->inv_scale = 1.0 / (double)rope_scale;
  r->log2_theta = std::log2((double)rope_theta);
  return PAGEDATTN_OK;
}

static int launch_rope_axes(const char* who, RopeAxesArgs r, bool bf16, bool append, bool fp8,
                            bool interleave, void* stream) {
  const int pairs = std::min(r.a.d / 16, kAxesFreqs / 8);
  r.c_shift = 0;
  while ((1 << r.c_shift) < pairs) ++r.c_shift;
  // tokens per workgroup: as many as one batch of loads covers, up to 4; one while
  // that makes two workgroups a CU or fewer (512 tokens of 8/1 heads, D = 128, 3.7
  // against 4.7 us with 4, of 32/4, D = 64, 3.7 against 5.2); and for many tokens of
  // few heads as many as leave four workgroups a CU, up to 16, which hide their
  // prologue better (8/1, D = 128: 8192 tokens 9.7 us with 8, 11.1 with 4; 65536 58.5
  // us with 16, 69.2 with 4; 4/1, D = 64, 65536 26.6 and 40.4).  12/2 heads, 128
  // lanes a token, gain less (65536 109.8 and 117.6, 4096 13.0 and 8.5) and stay
  // below the line.
  const int64_t lanes = ((int64_t)r.hq + (append ? 2 : 1) * (int64_t)r.a.hkv) << r.c_shift;
  const int64_t batch = kAxesThreads * kAxesBatch / 2 / std::max<int64_t>(lanes, 1);
  r.tokens = (int)std::max<int64_t>(
      1, std::min<int64_t>({4, batch, r.a.nnz / kAxesSpread}));
  if (lanes <= kAxesFewLanes)
    r.tokens = std::max(r.tokens, std::min(kAxesTokens, r.a.nnz / kAxesGroups));
  const dim3 grid((unsigned)(((int64_t)r.a.nnz + r.tokens - 1) / r.tokens),
                  (unsigned)((r.a.d / 16 + kAxesFreqs / 8 - 1) / (kAxesFreqs / 8)));
  auto* fn = bf16 ? (interleave ? pick_rope_axes<true, true>(append, fp8)
                                : pick_rope_axes<true, false>(append, fp8))
                  : (interleave ? pick_rope_axes<false, true>(append, fp8)
                                : pick_rope_axes<false, false>(append, fp8));
  hipLaunchKernelGGL(fn, grid, dim3(kAxesThreads), 0, (hipStream_t)stream, r);
  return check_launch(who);
}

}  // namespace pa

using namespace pa;

extern "C" {

int pagedattn_apply_multi_axis_rope_inplace(
    void* q, void* k, const int32_t* axis_positions, int64_t axis_stride, int32_t num_axes,
    const int32_t* sections, int32_t cyclic, int32_t nnz, int32_t num_qo_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t rotary_dim, int64_t q_stride_n,
    int64_t q_stride_h, int64_t k_stride_n, int64_t k_stride_h, int32_t interleave,
    float rope_scale, float rope_theta, int32_t dtype, void* stream) {
  const char* who = "apply_multi_axis_rope_inplace";
  if (dtype != PAGEDATTN_BF16 && dtype != PAGEDATTN_F16)
    return set_error(PAGEDATTN_ERR_UNSUPPORTED, "%s: dtype %d not supported (float16 or bfloat16)",
                     who, dtype);
  if (nnz < 0 || num_qo_heads < 0 || num_kv_heads < 0)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: bad shape nnz=%d hq=%d hkv=%d", who, nnz,
                     num_qo_heads, num_kv_heads);
  RopeAxesArgs r{};
  const int rc = axes_setup(who, axis_positions, axis_stride, num_axes, sections, cyclic, nnz,
                            head_dim, rotary_dim, rope_scale, rope_theta, &r);
  if (rc) return rc;
  if ((q_stride_n & 7) || (q_stride_h & 7) || (k_stride_n & 7) || (k_stride_h & 7) ||
      !aligned16(q) || !aligned16(k))
    return set_error(PAGEDATTN_ERR_UNSUPPORTED,
                     "%s: q and k must be 16-byte aligned with strides that are multiples of 8 "
                     "elements",
                     who);
  if (nnz == 0 || num_qo_heads + num_kv_heads == 0) return PAGEDATTN_OK;
  if ((num_qo_heads && !q) || (num_kv_heads && !k))
    return set_error(PAGEDATTN_ERR_INVALID, "%s: null pointer", who);
  r.a.k = static_cast<const uint16_t*>(k);
  r.a.k_sn = k_stride_n;
  r.a.k_sh = k_stride_h;
  r.a.nnz = nnz;
  r.a.hkv = num_kv_heads;
  r.a.d = head_dim;
  r.q = static_cast<uint16_t*>(q);
  r.q_sn = q_stride_n;
  r.q_sh = q_stride_h;
  r.hq = num_qo_heads;
  return launch_rope_axes(who, r, dtype == PAGEDATTN_BF16, false, false, interleave != 0, stream);
}

int pagedattn_multi_axis_rope_append_paged_kv_cache(
    void* q, int64_t q_stride_n, int64_t q_stride_h, int32_t num_qo_heads, void* append_key,
    const void* append_value, int64_t k_stride_n, int64_t k_stride_h, int64_t v_stride_n,
    int64_t v_stride_h, int32_t src_dtype, const int32_t* axis_positions, int64_t axis_stride,
    int32_t num_axes, const int32_t* sections, int32_t cyclic, const int32_t* batch_indices,
    const int32_t* positions, int32_t nnz, int32_t rotary_dim, int32_t interleave,
    float rope_scale, float rope_theta, void* paged_kv_cache, int32_t cache_dtype,
    const float* kv_scales, int32_t num_pages, const int32_t* kv_indices, int32_t num_indices,
    const int32_t* kv_indptr, int32_t batch_size, int32_t num_kv_heads, int32_t head_dim,
    int32_t page_size, int32_t* error_flag, void* stream) {
  const char* who = "multi_axis_rope_append_paged_kv_cache";
  if (num_qo_heads < 0)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: bad shape hq=%d", who, num_qo_heads);
  if ((q_stride_n & 7) || (q_stride_h & 7) || !aligned16(q))
    return set_error(PAGEDATTN_ERR_UNSUPPORTED,
                     "%s: q must be 16-byte aligned with strides that are multiples of 8 elements",
                     who);
  RopeAxesArgs r{};
  bool empty = false;
  int rc = append_setup(who, append_key, append_value, k_stride_n, k_stride_h, v_stride_n,
                        v_stride_h, src_dtype, batch_indices, positions, nnz, paged_kv_cache,
                        cache_dtype, kv_scales, num_pages, kv_indices, num_indices, kv_indptr,
                        batch_size, num_kv_heads, head_dim, page_size, error_flag, &r.a, &empty);
  if (!rc)
    rc = axes_setup(who, axis_positions, axis_stride, num_axes, sections, cyclic, nnz, head_dim,
                    rotary_dim, rope_scale, rope_theta, &r);
  if (rc || empty) return rc;
  if (num_qo_heads > 0 && !q) return set_error(PAGEDATTN_ERR_INVALID, "%s: null q", who);
  r.q = static_cast<uint16_t*>(q);
  r.q_sn = q_stride_n;
  r.q_sh = q_stride_h;
  r.hq = num_qo_heads;
  return launch_rope_axes(who, r, src_dtype == PAGEDATTN_BF16, true,
                          cache_dtype == PAGEDATTN_E4M3, interleave != 0, stream);
}

}  // extern "C"
