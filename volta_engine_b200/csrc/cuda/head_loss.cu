// Losses of a language model head without its logits: softmax cross entropy against labels, and KL(teacher || model) against a teacher's
// K most likely tokens and the mass of the rest; both with the gradients of the states and of the head.
//
//   z_rv = cap(sum_h x_rh W_vh),  cap(z) = c tanh(z / c) or z        s_rv = exp(z_rv - lse_r),  lse_r = log sum_v exp z_rv
//   cross entropy   nll_r = lse_r - z_ry = log(1 + exp(rest_r - z_ry))                     rest_r = log sum_{v != y} exp z_rv
//   divergence      kl_r  = sum_k a_k (log a_k - log s_k) + t (log t - log max(rho_r, 1e-12))    rho_r = exp(rest_r - lse_r), rest over v not in K
//   gradients       dz_rv = g_r s_rv ((A + t) - [v not in K] t / rho_r) - g_r [v in K] a_v,  A = sum_k a_k
//                   (the label is a teacher of one token: A = 1, t = 0; a likely one's own dz is taken as -g exp(rest - lse), which does not cancel)
//                   dx = (dz cap') W,  dW = (dz cap')^T x
//
// The logits exist a 256 x 256 tile at a time, in registers (gemm_pair.cuh). Scoring keeps of each row and 128 columns the maximum and the sum
// of exponentials without the targets, and the targets' logits; one more pass over these few numbers gives the loss. The targets are left
// out of the sums so that log(1 + exp(..)) and log(rho) do not come from the difference of two nearly equal numbers. The gradient computes the
// logits again, a piece of the vocabulary at a time, writes dz of that piece in bf16 slabs (rows x piece: the only array of that kind) and
// multiplies it with the head's rows and with the states. dz beside fp32 operands is three bf16 slabs (fp32's 24 bits), beside bf16 operands two
// (2^-16 of a value, and gradients are rounded to 2^-8 of theirs). One slab alone would be 2^-8 off as the gradients are, but of every addend: a row of dz
// sums to zero, so what the head's rows have in common leaves dx except for that rounding, and near a teacher the addends are far above their sum
// (errors of 2 to 6 times the gradients' own rounding; rows of dhead 1.3 to 2.9 times it).
// Sums run in a fixed order: the same call gives the same bits.
//
// Rows that are left out (label below zero, a teacher row of padding) are taken out in front: the states of the others are gathered, so what
// stands in the rest is never read, and time goes by the rows that count. The number of rows stays on the device.
#include "common.cuh"
#include "gemm_pair.cuh"
#include "tmap.h"

namespace ve {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLogFloor = -27.631021115928547f;       // log 1e-12: the least share of "any other token"
constexpr int kMaxTopk = 1024;
constexpr int kFrontRows = 4096, kFrontIds = 1 << 16;       // rows, or a teacher's ids, that every block of head_front_kernel looks through

VE_DEVINL float neg_inf() { return __int_as_float(0xff800000); }

// ------------------------------------------------------------------------------------------------ rows and operands
struct HeadRows {
  const void* labels;         // cross entropy: int32 or int64 [R]
  int label_bytes;
  const int* ids;             // divergence: [R, K]
  const float *logp, *tail;   // [R, K], [R]
  int K, R, V;
};

// Divergence: the teacher's tokens of a row in ascending order, with their places: sid / slp [R, K] (padding behind, as INT_MAX), and at
// off[r, b] the first one at or behind column span * b; flag[r]: the row counts; mass[r] = sum_k a_k.
struct TeacherRows {
  int span, nblk;
  int* sid;
  float* slp;
  uint16_t* off;
  int* flag;
  double* mass;
};
// One block (a multiple of 32 threads, at most 256) a row, counting ranks: K is small.
VE_DEVINL void sort_teacher(const HeadRows& p, const TeacherRows& o, int r) {
  __shared__ int id[kMaxTopk], srt[kMaxTopk];
  __shared__ double part[8];
  int any = 0;
  double sum = 0.0;
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
    const int v = p.ids[(size_t)r * p.K + k];
    id[k] = v < 0 ? INT_MAX : min(v, INT_MAX - 1);          // (any id behind the vocabulary is as wrong as the last)
    any |= v >= 0;
    if (v >= 0) sum += exp((double)p.logp[(size_t)r * p.K + k]);
  }
  for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  any = __syncthreads_or(any);
  if (threadIdx.x == 0) {
    double m = 0.0;
    for (int w = 0; w < (int)blockDim.x >> 5; ++w) m += part[w];
    o.flag[r] = any;
    o.mass[r] = m;
  }
  if (!any) return;                                   // (uniform)
  for (int k = threadIdx.x; k < p.K; k += blockDim.x) {
    const int v = id[k];
    int at = 0;
    for (int j = 0; j < p.K; ++j) at += id[j] < v || (id[j] == v && j < k);
    srt[at] = v;
    o.sid[(size_t)r * p.K + at] = v;
    o.slp[(size_t)r * p.K + at] = v == INT_MAX ? neg_inf() : p.logp[(size_t)r * p.K + k];
  }
  __syncthreads();
  for (int b = threadIdx.x; b <= o.nblk; b += blockDim.x) {
    int lo = 0, hi = p.K;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (srt[mid] < b * o.span) lo = mid + 1; else hi = mid;
    }
    o.off[(size_t)r * (o.nblk + 1) + b] = (uint16_t)lo;
  }
}
__global__ void __launch_bounds__(128) head_targets_kernel(const HeadRows p, const TeacherRows o) {
  grid_dep_launch();
  grid_dep_wait();
  sort_teacher(p, o, blockIdx.x);
}

VE_DEVINL long label_of(const HeadRows& p, int r) {
  return p.label_bytes == 8 ? (long)reinterpret_cast<const long long*>(p.labels)[r] : (long)reinterpret_cast<const int*>(p.labels)[r];
}

// Ranges of a piece's `steps` that dx is summed over: tiles x ranges fill whole waves of the 74 pairs; a range costs about 12 steps beside its products
// (its sums are written). Asked for on the device, where the number of rows that count is known: 819 of 2048 left half of the pairs idle.
struct DxPlan {
  int col_tiles, steps, pairs, most;
};
VE_DEVINL int dx_splits(int rows, const DxPlan& d) {
  const int tiles = (rows + 255) / 256 * d.col_tiles;
  int best = 1;
  float least = 0.f;
  for (int s = 1; s <= d.most && s * 4 <= d.steps; ++s) {
    const float cost = (float)((tiles * s + kPairClusters - 1) / kPairClusters) * (float)((d.steps + s - 1) / s * d.pairs + 12);
    if (s == 1 || cost < least) { least = cost; best = s; }
  }
  return best;
}

// The rows that count, in order: live[i] = row, pos[row] = i or -1, count[0] = their number, count[1] = ranges of dx.
__global__ void __launch_bounds__(1024) head_rows_kernel(const HeadRows p, const int* flag, int* live, int* pos, int* count, const DxPlan dx) {
  __shared__ int part[32], base;
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) base = 0;
  __syncthreads();
  for (int r0 = 0; r0 < p.R; r0 += 1024) {
    const int r = r0 + threadIdx.x;
    const bool on = r < p.R && (p.labels ? label_of(p, r) >= 0 : flag[r] != 0);
    const unsigned mask = __ballot_sync(0xffffffffu, on);
    if (lane == 0) part[warp] = __popc(mask);
    __syncthreads();
    int before = base;
    for (int w = 0; w < warp; ++w) before += part[w];
    const int at = before + __popc(mask & ((1u << lane) - 1));
    if (r < p.R) pos[r] = on ? at : -1;
    if (on) live[at] = r;
    __syncthreads();
    if (threadIdx.x == 1023) base = at + (on ? 1 : 0);
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    count[0] = base;
    count[1] = dx_splits(base, dx);
  }
}

// Eight values of a row from column c; zeros behind column H. `vec`: whole groups may be read as 16-byte words.
template <typename T>
VE_DEVINL void load8(const T* row, int c, int H, bool vec, float* v) {
  if (sizeof(T) == 4) {
    if (vec && c + 8 <= H) {
      const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < H ? (float)row[c + e] : 0.f;
    return;
  }
  uint32_t w[4];
  if (vec && c + 8 <= H) {
    const uint4 a = *reinterpret_cast<const uint4*>(row + c);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
  } else if (c + 8 <= H) {
    // a row that starts between 4-byte words: five words around its first and last value, which are inside the row's ends or beside them in their words
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + c);
    const uint32_t* q = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
    if (at & 2) {
      uint32_t x[5];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = q[e];
      x[4] = *reinterpret_cast<const unsigned short*>(q + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = __funnelshift_r(x[e], x[e + 1], 16);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = q[e];
    }
  } else {
    const unsigned short* s = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = (c + 2 * e < H ? s[c + 2 * e] : 0u) | (c + 2 * e + 1 < H ? (uint32_t)s[c + 2 * e + 1] << 16 : 0u);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) { v[2 * e] = __uint_as_float(w[e] << 16); v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
}

// Pairs of values to bf16, the values become what the rounding left (an infinity or a NaN leaves NaN).
VE_DEVINL uint32_t split_pair(float& lo, float& hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  const uint32_t b = *reinterpret_cast<const uint32_t*>(&v);
  lo -= __uint_as_float(b << 16);
  hi -= __uint_as_float(b & 0xffff0000u);
  return b;
}

// Columns [c0, c1) of a row (null: zeros) into its slabs, by a warp.
template <typename T>
VE_DEVINL void pack_row(const T* row, int c0, int c1, int H, int slabs, size_t slab, __nv_bfloat16* dst) {
  const bool vec = !(reinterpret_cast<uintptr_t>(row) & 15);
  for (int c = c0 + (threadIdx.x & 31) * 8; c < c1; c += 256) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row) load8(row, c, H, vec, v);
    for (int s = 0; s < slabs; ++s) {
      uint32_t b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = split_pair(v[2 * e], v[2 * e + 1]);
      *reinterpret_cast<uint4*>(dst + s * slab + c) = make_uint4(b[0], b[1], b[2], b[3]);
    }
  }
}

struct PackedRows {             // a matrix and its slabs [slabs][rows of a slab][Hp], zeros behind column H
  const void* src;
  long ld;
  int fp32, H, Hp, slabs;
  size_t slab;
  __nv_bfloat16* dst;
  VE_DEVINL int chunks() const { return (Hp + 255) >> 8; }
  VE_DEVINL void put(int row, bool there, int to, int chunk) const {        // row -> row `to` of the slabs, 256 columns, by a warp
    __nv_bfloat16* d = dst + (size_t)to * Hp;
    const int c0 = chunk * 256, c1 = min(Hp, c0 + 256);
    if (fp32) pack_row(there ? (const float*)src + row * ld : nullptr, c0, c1, H, slabs, slab, d);
    else pack_row(there ? (const __nv_bfloat16*)src + row * ld : nullptr, c0, c1, H, slabs, slab, d);
  }
};

// A warp a row. With `live`: the gathered rows, and zeros behind the last one to the end of its tile of 256 (the products along rows read them).
template <typename T>
__global__ void __launch_bounds__(256) head_pack_kernel(const PackedRows m, const int* live, const int* count, int rows) {
  grid_dep_launch();
  grid_dep_wait();
  const int n = live ? *count : rows, all = live ? (n + 255) / 256 * 256 : rows;
  for (int r = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < all; r += gridDim.x * blockDim.x >> 5)
    pack_row(r < n ? (const T*)m.src + (live ? live[r] : r) * m.ld : (const T*)nullptr, 0, m.Hp, m.H, m.slabs, m.slab, m.dst + (size_t)r * m.Hp);
}

// All of that for few rows in one launch: `teachers` blocks sort a teacher's row each; every other block finds all the rows that count and packs its
// share of them, and of the head where all of it is packed at once.
__global__ void __launch_bounds__(256) head_front_kernel(const HeadRows p, const TeacherRows teacher, int teachers, int* live, int* pos, int* count,
                                                         const PackedRows x, const PackedRows head, int head_rows, const DxPlan dx) {
  __shared__ int row_of[kFrontRows], part[8];
  grid_dep_launch();
  grid_dep_wait();
  if ((int)blockIdx.x < teachers) {
    sort_teacher(p, teacher, blockIdx.x);
    return;
  }
  const int block = blockIdx.x - teachers, blocks = gridDim.x - teachers;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // a thread looks at consecutive rows, 16 at most
  const int each = (p.R + 255) / 256, r0 = threadIdx.x * each;
  uint32_t mine = 0;
#pragma unroll 4
  for (int e = 0; e < each; ++e) {
    const int r = r0 + e;
    bool on = false;
    if (r < p.R) {
      if (p.labels) on = label_of(p, r) >= 0;
      else
        for (int k = 0; k < p.K && !on; k += 8)
#pragma unroll
          for (int g = 0; g < 8; ++g) on |= k + g < p.K && p.ids[(size_t)r * p.K + k + g] >= 0;
    }
    mine |= (uint32_t)on << e;
  }
  int at = __popc(mine), n = 0;
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, at, o);
    if (lane >= o) at += v;
  }
  if (lane == 31) part[warp] = at;
  at -= __popc(mine);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    if (w < warp) at += part[w];
    n += part[w];
  }
  for (int e = 0; e < each && r0 + e < p.R; ++e) {
    const bool on = mine >> e & 1u;
    if (on) row_of[at] = r0 + e;
    if (block == 0) {
      pos[r0 + e] = on ? at : -1;
      if (on) live[at] = r0 + e;
    }
    at += on;
  }
  __syncthreads();
  if (block == 0 && threadIdx.x == 0) {
    count[0] = n;
    count[1] = dx_splits(n, dx);
  }
  const int all = (n + 255) / 256 * 256, chunks = x.chunks();
  const size_t own = (size_t)all * chunks, units = own + (size_t)head_rows * chunks;
  for (size_t u = (size_t)block * 8 + warp; u < units; u += (size_t)blocks * 8) {
    const size_t v = u < own ? u : u - own;
    const int r = (int)(v / chunks), c = (int)(v - (size_t)r * chunks);
    if (u < own) x.put(r < n ? row_of[r] : 0, r < n, r, c);
    else head.put(r, true, r, c);
  }
}

// ------------------------------------------------------------------------------------------------ jobs of the paired GEMM
struct Targets {              // by row of the caller
  const void* labels;
  int label_bytes;
  const int* sid;             // [R, K]
  const float* slp;
  const uint16_t* off;        // [R, nblk + 1]
  int K, nblk;
  VE_DEVINL void range(int row, int blk, long col0, int cols, int& begin, int& end) const {      // targets of a row among a thread's columns
    if (labels) {
      const long y = label_bytes == 8 ? (long)reinterpret_cast<const long long*>(labels)[row] : (long)reinterpret_cast<const int*>(labels)[row];
      begin = 0;
      end = y >= col0 && y < col0 + cols;
    } else {
      const uint16_t* o = off + (size_t)row * (nblk + 1) + blk;
      begin = o[0];
      end = o[1];
    }
  }
  VE_DEVINL int id(int row, int p) const {
    if (labels) return label_bytes == 8 ? (int)reinterpret_cast<const long long*>(labels)[row] : reinterpret_cast<const int*>(labels)[row];
    return sid[(size_t)row * K + p];
  }
};

template <int C>              // columns of a thread
struct LogitTiles {           // rows x a piece of the vocabulary: tiles of up to 16 row tiles share the head's rows while L2 holds them
  static constexpr int NT = 2 * C;
  const int* count;
  int v0, nv, ksteps;
  VE_DEVINL int row_tiles() const { return (*count + 255) >> 8; }
  VE_DEVINL int tiles() const { return row_tiles() * ((nv + NT - 1) / NT); }
  struct Row { int row, begin, end, first; };        // the caller's row (-1: behind the last one), its targets among the thread's columns, the first one's column
  VE_DEVINL Row row_at(const PairTile& t, int r, int c0, const int* live, const Targets& tg) const {
    const int i = t.m0 + r, col0 = t.n0 + c0;
    Row w{i < *count ? live[i] : -1, 0, 0, -1};
    if (w.row >= 0 && col0 < nv) tg.range(w.row, (v0 + col0) / C, (long)v0 + col0, min(C, nv - col0), w.begin, w.end);
    if (w.begin < w.end) w.first = tg.id(w.row, w.begin) - v0 - col0;
    return w;
  }
  VE_DEVINL PairTile tile(int i) const {
    const int nm = row_tiles(), nn = (nv + NT - 1) / NT, per = 16 * nn;
    const int g = i / per, m_first = g * 16, gm = min(16, nm - m_first), j = i - g * per;
    return PairTile{(m_first + j % gm) * 256, (j / gm) * NT, 0, ksteps, 0};
  }
};

// A thread's logits through the cap. c tanh(z / c) = z f(x^2), x = z / c, with Lambert's continued fraction f = 1 / (1 + x^2 / (3 + x^2 / (5 + ..))) of
// tanh(x) / x; to seven terms it is 1.1e-8 off at x = 2 and less below. Where a lane's logits reach further the library's tanh is taken (128 of those
// are 5600 cycles a tile, these 1300).
template <bool CAP, int C>
VE_DEVINL void cap_logits(float* z, float cap, float inv_cap) {
  if (!CAP) return;
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < C; ++j) top = fmaxf(top, fabsf(z[j]));
  if (__any_sync(0xffffffffu, !(top <= 2.f * cap))) {
#pragma unroll
    for (int j = 0; j < C; ++j) z[j] = cap * tanhf(z[j] / cap);
  } else {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const float x = z[j] * inv_cap, y = x * x;
      const float num = fmaf(fmaf(y + 378.f, y, 17325.f), y, 135135.f), den = fmaf(fmaf(fmaf(28.f, y, 3150.f), y, 62370.f), y, 135135.f);
      z[j] *= num * rcp_approx(den);
    }
  }
}

template <bool CAP, int C>
struct ScoreJob : LogitTiles<C> {
  using Tiles = LogitTiles<C>;
  using Tiles::nv; using Tiles::v0;
  Targets tg;
  const int* live;
  int rows_cap;               // pitch of part
  float2* part;               // [block of C columns][row]: maximum and sum of exp(z - maximum) without the targets
  float* zt;                  // [R, K] logits of the targets, in the targets' ascending order
  float cap, inv_cap;
  using Row = typename Tiles::Row;
  VE_DEVINL Row begin(const PairTile& t, int r, int c0) const { return this->row_at(t, r, c0, live, tg); }

  VE_DEVINL void finish(const PairTile& t, int r, int c0, const Row& w, float* z, const CUtensorMap* omap, uint8_t* staging) const {
    const int i = t.m0 + r, row = w.row, col0 = t.n0 + c0, cols = min(C, nv - col0), blk = (v0 + col0) / C;
    if (!__any_sync(0xffffffffu, row >= 0) || cols <= 0) return;
    const bool on = row >= 0;
    int p = w.begin;
    const int end = w.end;
    cap_logits<CAP, C>(z, cap, inv_cap);
    if (cols < C) {
#pragma unroll
      for (int j = 0; j < C; ++j)
        if (j >= cols) z[j] = neg_inf();
    }
    // a token of each lane at a time: selects, for branches in the body of 128 columns fetch their code anew for every tile (20 us a tile that a target
    // falls into)
    int at = w.first;
    while (__any_sync(0xffffffffu, at >= 0)) {
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        v = j == at ? z[j] : v;
        z[j] = j == at ? neg_inf() : z[j];
      }
      if (at >= 0) {
        int next;
        do {                                        // (a token listed twice is one token)
          zt[(size_t)row * tg.K + p] = v;
          next = ++p < end ? tg.id(row, p) - v0 - col0 : -1;
        } while (next == at);
        at = next;
      }
    }
    float m = z[0];
#pragma unroll
    for (int j = 1; j < C; ++j) m = fmaxf(m, z[j]);
    const float m2 = m == neg_inf() ? 0.f : -(m * kLog2e);
    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
    for (int j = 0; j < C; j += 4) {
      s0 += ex2_approx(fmaf(z[j], kLog2e, m2));
      s1 += ex2_approx(fmaf(z[j + 1], kLog2e, m2));
      s2 += ex2_approx(fmaf(z[j + 2], kLog2e, m2));
      s3 += ex2_approx(fmaf(z[j + 3], kLog2e, m2));
    }
    // (what the product m log2e lost to rounding is in every term: 2^-18 of a sum beside logits of 100)
    if (on) part[(size_t)blk * rows_cap + i] = make_float2(m, ((s0 + s1) + (s2 + s3)) * exp2f(m == neg_inf() ? 0.f : -fmaf(m, kLog2e, m2)));
  }
};

// Constants of a row's dz: at any token dense * s, at a target `at` * s - g * (teacher's mass); a likely label's is `at` itself.
struct RowGrad {
  float lse2, dense, at, g;
};

struct RowInputs {            // by row of the caller
  const float *stats, *dloss, *tail;
  const double* mass;
  int R;
  bool labels, fine;          // fine: the statistics' lower parts stand behind them
  VE_DEVINL RowGrad at(int row) const {
    const double lse = (double)stats[row] + (fine ? (double)stats[2 * R + row] : 0.0), rest = (double)stats[R + row] + (fine ? (double)stats[3 * R + row] : 0.0);
    const float g = dloss[row];
    RowGrad c;
    // exp(z - lse) as 2^(z log2e - lse2): what the product lse log2e loses to rounding goes into the factors
    c.lse2 = (float)(lse * (double)kLog2e);
    const float fix = exp2f((float)((double)c.lse2 - lse * (double)kLog2e));
    c.g = g;
    if (labels) {
      c.dense = g * fix;
      c.at = -g * expf((float)(rest - lse));
    } else {
      const double a = mass[row], lr = rest - lse, t = lr >= (double)kLogFloor ? exp((double)tail[row]) : 0.0;
      c.at = (float)((double)g * (a + t)) * fix;
      c.dense = (float)((double)g * (t > 0.0 ? a + t - t * exp(-lr) : a)) * fix;       // (a difference: in 64 bits)
    }
    return c;
  }
};

template <bool CAP, int C>
struct GradJob : LogitTiles<C> {
  using Tiles = LogitTiles<C>;
  using Tiles::nv; using Tiles::v0;
  Targets tg;
  const int* live;
  RowInputs in;
  int slabs;                  // of dz
  static constexpr int kBox = C < 64 ? C : 64, kBoxes = C / kBox;        // columns that leave together
  float cap, inv_cap;

  struct Row : Tiles::Row {
    RowGrad c;
    float mass;               // the teacher's, of the first target
  };
  VE_DEVINL Row begin(const PairTile& t, int r, int c0) const {
    Row w{this->row_at(t, r, c0, live, tg), {0.f, 0.f, 0.f, 0.f}, 0.f};
    if (w.row >= 0) w.c = in.at(w.row);
    if (!tg.labels && w.first >= 0) w.mass = expf(tg.slp[(size_t)w.row * tg.K + w.begin]);
    return w;
  }

  VE_DEVINL void finish(const PairTile& t, int r, int c0, const Row& w, float* z, const CUtensorMap* omap, uint8_t* staging) const {
    const int i = t.m0 + r, row = w.row, end = w.end;
    const int col0 = t.n0 + c0, cols = max(0, min(C, nv - col0));
    const RowGrad c = w.c;
    int p = w.begin;
    // targets first, one of each lane at a time: their dz takes the logit's place, and its bit says that it stands there
    uint32_t set[C / 32] = {};
    cap_logits<CAP, C>(z, cap, inv_cap);
    int at = w.first;
    float mass = w.mass;
    const bool any = __any_sync(0xffffffffu, at >= 0);
    while (__any_sync(0xffffffffu, at >= 0)) {
      float v = 0.f, d = c.at;
#pragma unroll
      for (int j = 0; j < C; ++j) v = j == at ? z[j] : v;
      int next = -1;
      const float s = ex2_approx(fmaf(v, kLog2e, -c.lse2));
      if (tg.labels) {
        if (s < 0.5f) d = fmaf(c.dense, s, -c.g);          // (an unlikely label: s - 1 keeps what exp(rest - lse) loses to two roundings)
      } else if (at >= 0) {
        float a = mass;
        while (++p < end) {
          next = tg.id(row, p) - v0 - col0;
          mass = expf(tg.slp[(size_t)row * tg.K + p]);
          if (next != at) break;
          a += mass;
          next = -1;
        }
        d = fmaf(c.at, s, -c.g * a);
      }
      if (CAP) {
        const float th = v * inv_cap;
        d *= fmaf(-th, th, 1.f);
      }
#pragma unroll
      for (int k = 0; k < C / 32; ++k) set[k] |= at >> 5 == k ? 1u << (at & 31) : 0u;
#pragma unroll
      for (int j = 0; j < C; ++j) z[j] = j == at ? d : z[j];
      at = next;
    }
    const auto dz = [&](float v) {
      float f = c.dense;
      if (CAP) {
        const float th = v * inv_cap;
        f *= fmaf(-th, th, 1.f);
      }
      return f * ex2_approx(fmaf(v, kLog2e, -c.lse2));
    };
    if (any) {
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const float d = dz(z[j]);
        z[j] = set[j >> 5] >> (j & 31) & 1u ? z[j] : d;
      }
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j) z[j] = dz(z[j]);
    }
    if (__any_sync(0xffffffffu, row < 0 || cols < C)) {        // zeros to the ends of the tile: the products along rows and columns read them
      const int width = row >= 0 ? cols : 0;
#pragma unroll
      for (int j = 0; j < C; ++j) z[j] = j < width ? z[j] : 0.f;
    }
    for (int s = 0; s < slabs; ++s)
#pragma unroll
      for (int h = 0; h < kBoxes; ++h) {
        uint32_t b[kBox / 2];
#pragma unroll
        for (int j = 0; j < kBox / 2; ++j) b[j] = split_pair(z[kBox * h + 2 * j], z[kBox * h + 2 * j + 1]);
        put_box<false, 2 * kBox>(omap, staging, b, col0 + kBox * h, i & ~31, s);
      }
  }
};

// dx: gathered rows x H, along a piece of the vocabulary, cut into ranges that keep their own fp32 sums (the same number in every piece).
struct DxJob {
  const int* count;
  int H, Hp, ksteps, first;
  size_t slab;
  float* acc;                 // [ranges][rows_cap][Hp]
  struct Row {};
  VE_DEVINL Row begin(const PairTile&, int, int) const { return {}; }
  VE_DEVINL int row_tiles() const { return (*count + 255) >> 8; }
  VE_DEVINL int splits() const { return count[1]; }
  VE_DEVINL int tiles() const { return row_tiles() * ((H + 255) >> 8) * splits(); }
  VE_DEVINL PairTile tile(int i) const {
    const int nm = row_tiles(), tiles = nm * ((H + 255) >> 8), s = i / tiles, j = i - s * tiles;
    const int n = splits(), per = (ksteps + n - 1) / n;
    return PairTile{j % nm * 256, j / nm * 256, s * per, max(0, min(per, ksteps - s * per)), s};
  }
  VE_DEVINL void finish(const PairTile& t, int r, int c0, const Row& w, float* z, const CUtensorMap* omap, uint8_t* staging) const {
    const int x = t.n0 + c0, y = t.m0 + (r & ~31);
    if (y >= *count) return;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (x + 32 * g >= Hp) break;
      const uint32_t* b = reinterpret_cast<const uint32_t*>(z + 32 * g);
      // (one addition to each sum a piece, the pieces in order: no choice of order; waiting for the old sums took 17 % of a piece)
      if (first) put_box<false>(omap, staging, b, x + 32 * g, y, t.split);
      else put_box<true>(omap, staging, b, x + 32 * g, y, t.split);
    }
  }
};

// dW: a piece of the vocabulary x H, along the gathered rows.
template <typename T>
struct DheadJob {
  const int* count;
  int nv, H;
  T* out;                     // [nv, H], contiguous rows
  bool boxes;                 // rows on 16-byte boundaries: written by TMA (omap)
  static constexpr int kBox = 128 / sizeof(T);
  struct Row {};
  VE_DEVINL Row begin(const PairTile&, int, int) const { return {}; }
  VE_DEVINL int tiles() const { return ((nv + 255) >> 8) * ((H + 255) >> 8); }
  VE_DEVINL PairTile tile(int i) const {
    const int nn = (H + 255) >> 8;
    return PairTile{i / nn * 256, i % nn * 256, 0, (*count + 63) >> 6, 0};
  }
  VE_DEVINL void finish(const PairTile& t, int r, int c0, const Row& w, float* z, const CUtensorMap* omap, uint8_t* staging) const {
    const int cols = H - t.n0 - c0;
    if (cols <= 0 || t.m0 + (r & ~31) >= nv) return;
    if (boxes) {
#pragma unroll
      for (int g = 0; g < 128 / kBox; ++g) {
        if (g * kBox >= cols) break;
        uint32_t b[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) b[j] = sizeof(T) == 4 ? __float_as_uint(z[32 * g + j]) : split_pair(z[kBox * g + 2 * j], z[kBox * g + 2 * j + 1]);
        put_box<false>(omap, staging, b, t.n0 + c0 + kBox * g, t.m0 + (r & ~31), 0);
      }
      return;
    }
    // rows off 16-byte boundaries: 32 x 32 values at a time through shared memory, so that a warp writes along a row (a thread along its own: 45 us
    // where this takes 14, 5003 x 515)
    const int lane = threadIdx.x & 31;
    float* st = reinterpret_cast<float*>(staging);
    const int v0 = t.m0 + (r & ~31);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
#pragma unroll
      for (int j = 0; j < 32; ++j) st[lane * 32 + (j ^ lane)] = z[32 * g + j];
      __syncwarp();
      const int c = 32 * g + lane;
      if (c < cols)
        for (int k = 0; k < 32 && v0 + k < nv; ++k) out[(size_t)(v0 + k) * H + t.n0 + c0 + c] = (T)st[k * 32 + (lane ^ k)];
      __syncwarp();
    }
  }
};

template <int NT, bool A_MN, bool B_MN, bool ONE, class Job>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
head_gemm_kernel(const Job job, const PairLoop loop, const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                 const __grid_constant__ CUtensorMap omap, int* status) {
  grid_dep_launch();
  pair_gemm<NT, A_MN, B_MN, ONE>(job, loop, &amap, &bmap, &omap, status, [] { grid_dep_wait(); });
}

// ------------------------------------------------------------------------------------------------ the rows' sums
// Joins a row's blocks and computes its loss, 32 rows a block of 1024 threads: the warps share the blocks of columns, lanes are rows; then a
// warp takes a row's targets. The few numbers behind the sums are in 64 bits: losses near zero, and divergences of near models, are differences.
__global__ void __launch_bounds__(1024) head_merge_kernel(const HeadRows p, const int* live, const int* pos, const int* count, int rows_cap, int nblk,
                                                          const float2* part, const float* zt, const int* sid, const float* slp, float* loss, float* stats, int fine) {
  __shared__ float sm[32][33], ss[32][33];
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = *count;
  const int r = blockIdx.x * 32 + lane;
  if (warp == 0 && r < p.R && pos[r] < 0) {          // left out
    loss[r] = stats[r] = stats[p.R + r] = 0.f;
    if (fine) stats[2 * p.R + r] = stats[3 * p.R + r] = 0.f;
  }
  if (blockIdx.x * 32 >= n) return;
  const int i = blockIdx.x * 32 + lane;
  float m = neg_inf(), s = 0.f;
  if (i < n) {
    for (int b0 = warp; b0 < nblk; b0 += 32 * 8) {
      float2 v[8];
      float mx = m;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int b = b0 + 32 * e;
        v[e] = b < nblk ? part[(size_t)b * rows_cap + i] : make_float2(neg_inf(), 0.f);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, v[e].x);
      // (maxima pass NaN over, sums keep it: a block of NaN alone has a maximum of minus infinity or NaN, and counts)
      const float at = mx == neg_inf() ? 0.f : mx;
      s *= exp2f((m - at) * kLog2e);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[e].y * exp2f((v[e].x - at) * kLog2e);
      m = mx;
    }
  }
  sm[warp][lane] = m;
  ss[warp][lane] = s;
  __syncthreads();
  const int j = blockIdx.x * 32 + warp;               // this warp's row
  if (j >= n) return;
  const float wm = sm[lane][warp];
  const float top = warp_max(wm);
  const double sum = [&] {
    double v = (double)ss[lane][warp] * exp2((double)(wm - (top == neg_inf() ? 0.f : top)) * 1.4426950408889634);
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }();
  const int row = live[j];
  const double rest = (double)top + log(sum);          // (no token besides the targets: minus infinity)
  double lse, out;
  if (p.labels) {
    const long y = label_of(p, row);
    const double z = zt[row], d = rest - z;
    out = d > 0 ? d + log1p(exp(-d)) : log1p(exp(d));
    lse = z + out;
    if (y >= p.V) out = lse = __longlong_as_double(0x7ff8000000000000ll);
  } else {
    const int* id = sid + (size_t)row * p.K;
    const float* z = zt + (size_t)row * p.K;
    const float* lp = slp + (size_t)row * p.K;
    // sum over the targets: each token once
    double mx = rest;
    bool bad = false;
    for (int k = lane; k < p.K; k += 32) {
      bad |= id[k] >= p.V && id[k] != INT_MAX;
      if (id[k] < p.V) mx = fmax(mx, (double)z[k]);
    }
    for (int o = 16; o > 0; o >>= 1) mx = fmax(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    double v = 0.0;
    for (int k = lane; k < p.K; k += 32)
      if (id[k] < p.V && (k == 0 || id[k - 1] != id[k])) v += exp((double)z[k] - mx);
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    lse = mx + log(v + (rest == -INFINITY ? 0.0 : exp(rest - mx)));
    out = 0.0;
    for (int k = lane; k < p.K; k += 32) {
      if (id[k] >= p.V || (k > 0 && id[k - 1] == id[k])) continue;
      double a = exp((double)lp[k]), la = lp[k];
      if (k + 1 < p.K && id[k + 1] == id[k]) {          // (listed again: its mass is the sum)
        for (int j = k + 1; j < p.K && id[j] == id[k]; ++j) a += exp((double)lp[j]);
        la = log(a);
      }
      if (a != 0.0) out += a * (la - ((double)z[k] - lse));
    }
    for (int o = 16; o > 0; o >>= 1) out += __shfl_xor_sync(0xffffffffu, out, o);
    const float lt = p.tail[row];
    if (lt != neg_inf()) out += exp((double)lt) * ((double)lt - fmax(rest - lse, (double)kLogFloor));
    if (__any_sync(0xffffffffu, bad)) out = lse = __longlong_as_double(0x7ff8000000000000ll);
  }
  if (lane == 0) {
    loss[row] = (float)out;
    stats[row] = (float)lse;
    stats[p.R + row] = (float)rest;
    if (fine) {          // what the rounding left
      stats[2 * p.R + row] = isinf(lse) ? 0.f : (float)(lse - (double)(float)lse);
      stats[3 * p.R + row] = isinf(rest) ? 0.f : (float)(rest - (double)(float)rest);
    }
  }
}

// dx of the caller's rows from the ranges' sums; zeros where a row was left out.
template <typename T>
__global__ void __launch_bounds__(256) head_dx_kernel(const DxJob job, const int* pos, int R, T* dx) {
  grid_dep_launch();
  grid_dep_wait();
  const int H = job.H, Hp = job.Hp, splits = job.splits();
  const int per = (H + 3) / 4;
  const bool vec = !((uintptr_t)dx & 15) && H % 4 == 0;
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < (size_t)R * per; i += (size_t)gridDim.x * blockDim.x) {
    const int r = (int)(i / per), c = (int)(i - (size_t)r * per) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    const int at = pos[r];
    if (at >= 0) {
      const float* a = job.acc + (size_t)at * Hp + c;
      for (int s = 0; s < splits; ++s) {
        const float4 w = *reinterpret_cast<const float4*>(a + s * job.slab);
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
      }
    }
    T* dst = dx + (size_t)r * H + c;
    const T o[4] = {(T)v.x, (T)v.y, (T)v.z, (T)v.w};
    if (vec) {
      if (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(o);
      else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < H) dst[e] = o[e];
    }
  }
}

// ------------------------------------------------------------------------------------------------ host side
struct HeadPlan {             // sizes and places in the workspace
  int Hp, sx, sw, sg;         // padded width; slabs of the states, the head, dz
  int rows_cap, ksteps;
  int span, nblk;             // columns of a thread of the logits' tiles, and blocks of so many in the vocabulary
  bool few;                   // rows that one launch looks through and packs
  bool pack_head;             // the head's rows go through slabs of their own, a piece at a time
  int piece;                  // vocabulary rows at a time
  int splits, pairs;          // most ranges of a piece that dx is summed over; products of slabs
  size_t live, pos, count, flag, mass, sid, slp, off, x, part, zt, head, G, acc, bytes;
};

static inline int blocks_of(size_t n, int per = 256) {
  const size_t b = (n + per - 1) / per;
  return (int)(b < 148 * 16 ? (b ? b : 1) : 148 * 16);
}

// Sizes of pieces: dz of a piece takes 256 MB at most, packed rows of the head 512 MB (pieces that stay in L2 are slower: 1 x 838 x 77594 in fp32 378 us
// at 64 MB, 295 at 512: short waves).
static HeadPlan head_plan(bool grads, bool want_dx, int x_fp32, int head_fp32, bool pack_head, int R, int H, int V, int K, bool kl) {
  HeadPlan p;
  p.Hp = (H + 7) / 8 * 8;
  p.sx = x_fp32 ? 3 : 1;
  p.sw = head_fp32 ? 3 : 1;
  p.sg = x_fp32 || head_fp32 ? 3 : 2;
  p.rows_cap = (R + 255) / 256 * 256;
  size_t piece = ((size_t)V + 255) / 256 * 256;
  if (pack_head) { const size_t most = (512ull << 20) / ((size_t)p.sw * p.Hp * 2) / 256 * 256; piece = piece < most ? piece : (most ? most : 256); }
  if (grads) { const size_t most = (256ull << 20) / ((size_t)p.sg * p.rows_cap * 2) / 256 * 256; piece = piece < most ? piece : (most ? most : 256); }
  p.piece = (int)piece;
  // tiles of 256 columns where they give every pair one, otherwise of 64 (96 x 512 x 4099 in fp32 with gradients 89 us against 99, 77 x 515 x 5003 with a
  // teacher and a cap 84 against 96)
  p.span = (long)(p.rows_cap / 256) * (p.piece / 256) < kPairClusters ? 32 : 128;
  p.nblk = (V + p.span - 1) / p.span;
  p.ksteps = (H + 63) / 64;
  p.pack_head = pack_head;
  p.few = R <= kFrontRows && (!kl || (size_t)R * K <= kFrontIds);
  p.pairs = x_fp32 ? (head_fp32 ? 6 : 3) : (head_fp32 ? 3 : 2);
  const size_t sums = 4ull * p.rows_cap * p.Hp;                                          // of a range of dx: 256 MB together
  p.splits = (int)((256ull << 20) / sums < 1 ? 1 : (256ull << 20) / sums < 32 ? (256ull << 20) / sums : 32);
  size_t at = 0;
  auto take = [&](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
  p.live = take(4ull * R); p.pos = take(4ull * R); p.count = take(8);
  p.flag = p.mass = p.sid = p.slp = p.off = 0;
  if (kl) { p.flag = take(4ull * R); p.mass = take(8ull * R); p.sid = take(4ull * R * K); p.slp = take(4ull * R * K); p.off = take(2ull * R * (p.nblk + 1)); }
  p.x = take(2ull * p.sx * p.rows_cap * p.Hp);
  p.head = pack_head ? take(2ull * p.sw * p.piece * p.Hp) : 0;
  p.part = p.zt = p.G = p.acc = 0;
  if (!grads) { p.part = take(8ull * p.nblk * p.rows_cap); p.zt = take(4ull * R * (kl ? K : 1)); }
  else {
    p.G = take(2ull * p.sg * p.rows_cap * p.piece);
    if (want_dx) p.acc = take(4ull * p.splits * p.rows_cap * p.Hp);
  }
  p.bytes = at;
  return p;
}

struct HeadCall {
  const void* x; int x_fp32; long ldx;
  const void* head; int head_fp32; long ldw;
  HeadRows rows;
  int H;
  float softcap;
  uint8_t* ws;
  int* status;
  cudaStream_t st;
};

static bool head_packs(const void* head, int head_fp32, long ldw, int H) { return head_fp32 || H % 8 || ldw % 8 || ((uintptr_t)head & 15); }

// Boxes of 64 columns and 128 or 32 rows (an operand along its columns) or 64 rows (one along its rows).
static int slab_map(CUtensorMap* m, const void* base, int slabs, uint64_t slab_rows, uint64_t rows, uint64_t cols, uint64_t pitch, int box_rows) {
  return make_tmap_3d(m, base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, slabs, rows, cols, slab_rows * pitch * 2, pitch * 2, box_rows, 64, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int NT, bool A_MN, bool B_MN, bool ONE, class Job>
static int launch_pair_as(const Job& job, const PairLoop& loop, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o, const HeadCall& c) {
  cudaError_t e = allow_smem<head_gemm_kernel<NT, A_MN, B_MN, ONE, Job>>(kPairSmem);
  if (e != cudaSuccess) return (int)e;
  launch_pdl(head_gemm_kernel<NT, A_MN, B_MN, ONE, Job>, dim3(2 * kPairClusters), dim3(kPairThreads), kPairSmem, c.st, job, loop, a, b, o, c.status);
  return (int)cudaGetLastError();
}
template <int NT, bool A_MN, bool B_MN, class Job>
static int launch_pair(const Job& job, const PairLoop& loop, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o, const HeadCall& c) {
  return loop.na * loop.nb == 1 ? launch_pair_as<NT, A_MN, B_MN, true>(job, loop, a, b, o, c) : launch_pair_as<NT, A_MN, B_MN, false>(job, loop, a, b, o, c);
}

static PackedRows states_of(const HeadCall& c, const HeadPlan& p) {
  return PackedRows{c.x, c.ldx, c.x_fp32, c.H, p.Hp, p.sx, (size_t)p.rows_cap * p.Hp, (__nv_bfloat16*)(c.ws + p.x)};
}
static PackedRows head_of(const HeadCall& c, const HeadPlan& p, int v0) {
  const size_t es = c.head_fp32 ? 4 : 2;
  return PackedRows{(const uint8_t*)c.head + (size_t)v0 * c.ldw * es, c.ldw, c.head_fp32, c.H, p.Hp, p.sw, (size_t)p.piece * p.Hp, (__nv_bfloat16*)(c.ws + p.head)};
}
// (a large head is packed by a launch of its own, whose blocks have nothing else to do: 100 MB take 33 us there and 40 in front)
static bool head_in_front(const HeadCall& c, const HeadPlan& p) { return p.pack_head && p.few && p.piece >= c.rows.V && (size_t)c.rows.V * p.Hp <= 4u << 20; }
static int pack_blocks(const HeadPlan& p, size_t rows) { return blocks_of(rows * ((p.Hp + 255) / 256), 8); }
static void pack_rows(const PackedRows& m, const int* live, const int* count, int rows, cudaStream_t st) {
  const dim3 grid(blocks_of((size_t)rows, 8));
  if (m.fp32) launch_pdl(head_pack_kernel<float>, grid, dim3(256), 0, st, m, live, count, rows);
  else launch_pdl(head_pack_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, m, live, count, rows);
}

// The rows that count, their targets and their states; a head that is packed at once.
static int head_front(const HeadCall& c, const HeadPlan& p) {
  int *live = (int*)(c.ws + p.live), *pos = (int*)(c.ws + p.pos), *count = (int*)(c.ws + p.count), *flag = (int*)(c.ws + p.flag);
  const TeacherRows teacher{p.span, p.nblk, (int*)(c.ws + p.sid), (float*)(c.ws + p.slp), (uint16_t*)(c.ws + p.off), flag, (double*)(c.ws + p.mass)};
  const DxPlan dx{(c.H + 255) / 256, p.piece / 64, p.pairs, p.acc ? p.splits : 0};
  const int R = c.rows.R, teachers = c.rows.labels ? 0 : R;
  if (p.few) {
    const int heads = head_in_front(c, p) ? c.rows.V : 0;
    launch_pdl(head_front_kernel, dim3(teachers + pack_blocks(p, (size_t)p.rows_cap + heads)), dim3(256), 0, c.st, c.rows, teacher, teachers, live, pos, count,
               states_of(c, p), head_of(c, p, 0), heads, dx);
    return (int)cudaGetLastError();
  }
  if (teachers) launch_pdl(head_targets_kernel, dim3(R), dim3(128), 0, c.st, c.rows, teacher);
  launch_pdl(head_rows_kernel, dim3(1), dim3(1024), 0, c.st, c.rows, (const int*)flag, live, pos, count, dx);
  pack_rows(states_of(c, p), live, count, R, c.st);
  return (int)cudaGetLastError();
}

// The head's rows [v0, v0 + nv) as an operand: in place, or packed.
static int head_rows_map(CUtensorMap* m, const HeadCall& c, const HeadPlan& p, int v0, int nv, int box_rows, bool pack) {
  if (!p.pack_head) return slab_map(m, (const __nv_bfloat16*)c.head + (size_t)v0 * c.ldw, 1, nv, nv, c.H, c.ldw, box_rows);
  if (pack && !head_in_front(c, p))
    pack_rows(head_of(c, p, v0), nullptr, nullptr, nv, c.st);
  return slab_map(m, c.ws + p.head, p.sw, p.piece, nv, p.Hp, p.Hp, box_rows);
}

static Targets head_targets_of(const HeadCall& c, const HeadPlan& p) {
  return Targets{c.rows.labels, c.rows.label_bytes, (const int*)(c.ws + p.sid), (const float*)(c.ws + p.slp), (const uint16_t*)(c.ws + p.off),
                 c.rows.labels ? 1 : c.rows.K, p.nblk};
}

// Steps of 64 between fp32 additions where 32 bits are asked for. Cut-off sums over a step are 5e-8 too small; this keeps that below what fp32 additions
// along H round by (H = 128 7e-8, 1024 2.5e-7, 5120 7e-7). Shorter pieces wait for their additions: of one step 15 to 50 %, of two up to 6 %. Steps of
// several slabs are long enough to be pieces by themselves.
static inline int exact_chunk(int sa, int sb, int H) { return sa * sb > 1 ? 1 : H <= 256 ? 1 : H <= 640 ? 2 : 4; }
// Where the result is rounded to bf16 (cut-off sums over 2048: 2e-6): about 32 steps of one pair.
static inline PairLoop rounded_loop(int sa, int sb) {
  PairLoop l = pair_loop(sa, sb, 1, 32);
  l.chunk = 32 / l.pairs;
  return l;
}
static inline PairLoop exact_loop(int sa, int sb, int H) { return pair_loop(sa, sb, 2, exact_chunk(sa, sb, H)); }

template <bool CAP, int C>
static int head_score(const HeadCall& c, const HeadPlan& p, float* loss, float* stats, int fine) {
  int rc = head_front(c, p);
  if (rc) return rc;
  const int *live = (const int*)(c.ws + p.live), *pos = (const int*)(c.ws + p.pos), *count = (const int*)(c.ws + p.count);
  CUtensorMap xm, wm;
  rc = slab_map(&xm, c.ws + p.x, p.sx, p.rows_cap, p.rows_cap, p.Hp, p.Hp, 128);
  if (rc) return rc;
  ScoreJob<CAP, C> job;
  job.count = count; job.ksteps = p.ksteps; job.tg = head_targets_of(c, p); job.live = live; job.rows_cap = p.rows_cap;
  job.part = (float2*)(c.ws + p.part); job.zt = (float*)(c.ws + p.zt); job.cap = c.softcap; job.inv_cap = CAP ? 1.f / c.softcap : 0.f;
  for (int v0 = 0; v0 < c.rows.V; v0 += p.piece) {
    job.v0 = v0;
    job.nv = c.rows.V - v0 < p.piece ? c.rows.V - v0 : p.piece;
    if ((rc = head_rows_map(&wm, c, p, v0, job.nv, C, true))) return rc;
    if ((rc = launch_pair<2 * C, false, false>(job, exact_loop(p.sx, p.sw, c.H), xm, wm, xm, c))) return rc;
  }
  launch_pdl(head_merge_kernel, dim3((c.rows.R + 31) / 32), dim3(1024), 0, c.st, c.rows, live, pos, count, p.rows_cap, p.nblk, (const float2*)job.part,
             (const float*)job.zt, job.tg.sid, job.tg.slp, loss, stats, fine);
  return (int)cudaGetLastError();
}

template <bool CAP, int C>
static int head_grad(const HeadCall& c, const HeadPlan& p, const float* stats, int fine, const float* dloss, void* dx, void* dhead) {
  int rc = head_front(c, p);
  if (rc) return rc;
  const int *live = (const int*)(c.ws + p.live), *pos = (const int*)(c.ws + p.pos), *count = (const int*)(c.ws + p.count);
  const int R = c.rows.R, H = c.H;
  GradJob<CAP, C> gj;
  CUtensorMap xk, xmn, wk, wmn, gk, gmn, gout, aout, hout;
  rc = slab_map(&xk, c.ws + p.x, p.sx, p.rows_cap, p.rows_cap, p.Hp, p.Hp, 128);
  if (!rc) rc = slab_map(&xmn, c.ws + p.x, p.sx, p.rows_cap, p.rows_cap, p.Hp, p.Hp, 64);
  if (!rc) rc = slab_map(&gk, c.ws + p.G, p.sg, p.rows_cap, p.rows_cap, p.piece, p.piece, 128);
  if (!rc) rc = slab_map(&gmn, c.ws + p.G, p.sg, p.rows_cap, p.rows_cap, p.piece, p.piece, 64);
  if (!rc && dx)
    rc = make_tmap_3d(&aout, c.ws + p.acc, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, p.splits, p.rows_cap, p.Hp, 4ull * p.rows_cap * p.Hp, 4ull * p.Hp, 32, 32,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc)
    rc = make_tmap_3d(&gout, c.ws + p.G, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.sg, p.rows_cap, p.piece, 2ull * p.rows_cap * p.piece, 2ull * p.piece, 32,
                      gj.kBox, gj.kBox == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
  if (rc) return rc;
  gj.count = count; gj.ksteps = p.ksteps; gj.tg = head_targets_of(c, p); gj.live = live;
  gj.slabs = p.sg; gj.cap = c.softcap; gj.inv_cap = CAP ? 1.f / c.softcap : 0.f;
  gj.in = RowInputs{stats, dloss, c.rows.tail, (const double*)(c.ws + p.mass), R, c.rows.labels != nullptr, fine != 0};
  DxJob xj{count, H, p.Hp, 0, 1, (size_t)p.rows_cap * p.Hp, (float*)(c.ws + p.acc)};
  // the logits are summed in the scored ones' steps: beside an lse of exacter sums, 2e-6 of z are errors of s that a row has in common (rows whose model
  // is near its teacher or label: up to 6 times the gradients' rounding, 60 x 4096 x 5000; here 2 to 3 % of the time)
  for (int v0 = 0; v0 < c.rows.V; v0 += p.piece) {
    const int nv = c.rows.V - v0 < p.piece ? c.rows.V - v0 : p.piece;
    gj.v0 = v0;
    gj.nv = nv;
    if ((rc = head_rows_map(&wk, c, p, v0, nv, C, true))) return rc;
    if ((rc = launch_pair<2 * C, false, false>(gj, exact_loop(p.sx, p.sw, c.H), xk, wk, gout, c))) return rc;
    if (dx) {
      if ((rc = head_rows_map(&wmn, c, p, v0, nv, 64, false))) return rc;
      xj.ksteps = (nv + 63) / 64;
      xj.first = v0 == 0;
      const PairLoop loop = c.x_fp32 ? exact_loop(p.sg, p.sw, 1 << 30) : rounded_loop(p.sg, p.sw);
      if ((rc = launch_pair_as<256, false, true, false>(xj, loop, gk, wmn, aout, c))) return rc;
    }
    if (dhead) {
      const size_t es = c.head_fp32 ? 4 : 2;
      uint8_t* out = (uint8_t*)dhead + (size_t)v0 * H * es;
      const bool boxes = H * es % 16 == 0 && !((uintptr_t)dhead & 15);
      if (boxes && (rc = make_tmap_3d(&hout, out, c.head_fp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (int)es, 1, nv, H, (uint64_t)nv * H * es,
                                      H * es, 32, (uint32_t)(128 / es), CU_TENSOR_MAP_SWIZZLE_128B)))
        return rc;
      if (!boxes) hout = gmn;
      if (c.head_fp32) {
        const DheadJob<float> job{count, nv, H, (float*)out, boxes};
        rc = launch_pair_as<256, true, true, false>(job, exact_loop(p.sg, p.sx, 1 << 30), gmn, xmn, hout, c);
      } else {
        const DheadJob<__nv_bfloat16> job{count, nv, H, (__nv_bfloat16*)out, boxes};
        rc = launch_pair_as<256, true, true, false>(job, rounded_loop(p.sg, p.sx), gmn, xmn, hout, c);
      }
      if (rc) return rc;
    }
  }
  if (dx) {
    const int grid = blocks_of((size_t)R * p.Hp / 4);
    if (c.x_fp32) launch_pdl(head_dx_kernel<float>, dim3(grid), dim3(256), 0, c.st, xj, pos, R, (float*)dx);
    else launch_pdl(head_dx_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, c.st, xj, pos, R, (__nv_bfloat16*)dx);
  }
  return (int)cudaGetLastError();
}

}  // namespace ve

using namespace ve;

extern "C" {

// Bytes of workspace that a call needs (256-byte aligned). packs: the head is fp32, or its width, pitch or start keep its rows off 16-byte boundaries.
long ve_head_loss_workspace(int grads, int want_dx, int x_fp32, int head_fp32, int packs, int R, int H, int V, int K, int kl) {
  return (long)head_plan(grads, want_dx, x_fp32, head_fp32, packs, R, H, V, K, kl).bytes;
}

// x [R, H] (row pitch ldx), head [V, H] (pitch ldw), each bf16 or fp32. labels (int32 / int64 [R]) or ids int32 [R, K] with logp fp32 [R, K] and
// tail fp32 [R]. loss fp32 [R], stats fp32 [2, R]: log sum exp of all logits, and of all but the targets; fine: [4, R], what rounding both to 32 bits left
// behind them.
int ve_head_loss(const void* x, int x_fp32, long ldx, const void* head, int head_fp32, long ldw, const void* labels, int label_bytes, const void* ids,
                 const void* logp, const void* tail, int K, int R, int H, int V, float softcap, void* loss, void* stats, int fine, void* ws, long ws_bytes, void* status,
                 cudaStream_t st) {
  if (R <= 0) return 0;
  if (H <= 0 || V <= 0 || (!labels && (K < 1 || K > kMaxTopk))) return cudaErrorInvalidValue;
  const HeadPlan p = head_plan(false, false, x_fp32, head_fp32, head_packs(head, head_fp32, ldw, H), R, H, V, K, !labels);
  if ((size_t)ws_bytes < p.bytes) return cudaErrorInvalidValue;
  const HeadCall c{x, x_fp32, ldx, head, head_fp32, ldw, {labels, label_bytes, (const int*)ids, (const float*)logp, (const float*)tail, K, R, V}, H, softcap,
                   (uint8_t*)ws, (int*)status, st};
  if (p.span == 32) return softcap > 0.f ? head_score<true, 32>(c, p, (float*)loss, (float*)stats, fine) : head_score<false, 32>(c, p, (float*)loss, (float*)stats, fine);
  return softcap > 0.f ? head_score<true, 128>(c, p, (float*)loss, (float*)stats, fine) : head_score<false, 128>(c, p, (float*)loss, (float*)stats, fine);
}

// The gradients for dloss fp32 [R]: dx [R, H] in the states' type and dhead [V, H] in the head's, either may be null.
int ve_head_loss_grad(const void* x, int x_fp32, long ldx, const void* head, int head_fp32, long ldw, const void* labels, int label_bytes, const void* ids,
                      const void* logp, const void* tail, int K, int R, int H, int V, float softcap, const void* stats, int fine, const void* dloss, void* dx, void* dhead,
                      void* ws, long ws_bytes, void* status, cudaStream_t st) {
  if (R <= 0 || (!dx && !dhead)) return 0;
  if (H <= 0 || V <= 0 || (!labels && (K < 1 || K > kMaxTopk))) return cudaErrorInvalidValue;
  const HeadPlan p = head_plan(true, dx != nullptr, x_fp32, head_fp32, head_packs(head, head_fp32, ldw, H), R, H, V, K, !labels);
  if ((size_t)ws_bytes < p.bytes) return cudaErrorInvalidValue;
  const HeadCall c{x, x_fp32, ldx, head, head_fp32, ldw, {labels, label_bytes, (const int*)ids, (const float*)logp, (const float*)tail, K, R, V}, H, softcap,
                   (uint8_t*)ws, (int*)status, st};
  const float *s = (const float*)stats, *g = (const float*)dloss;
  if (p.span == 32) return softcap > 0.f ? head_grad<true, 32>(c, p, s, fine, g, dx, dhead) : head_grad<false, 32>(c, p, s, fine, g, dx, dhead);
  return softcap > 0.f ? head_grad<true, 128>(c, p, s, fine, g, dx, dhead) : head_grad<false, 128>(c, p, s, fine, g, dx, dhead);
}

}  // extern "C"
