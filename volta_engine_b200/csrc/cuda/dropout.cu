// Dropout with an added residual; the mask is computed where it is needed and never stored:
//   y[r, c] = residual[r, c] + keep(r, c) x[r, c] scale,    dx[r, c] = keep(r, c) dy[r, c] scale,    scale = 65536 / (65536 - t)
//
// keep(r, c): 16 bits of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) at counter
// (c / 8, row low, row high, site) and key seed, row = row0 + r; element c takes half c % 8 of the four words (word c % 8 / 2, low half first) and
// is kept if that half is at least t. t = p * 65536 rounded: p is met to 2^-17, the scale fits the t that is used. A mask bit depends on nothing but
// (seed, site, row, column): a checkpointed layer that runs again, the backward pass and a rank that holds some of the rows all compute the same one.
//
// One read of x (and residual) and one write: bound by memory, 16384 x 5120 bf16 with residual 76 us (6.6 TB/s), its gradient 64 us (5.3 TB/s: fewer
// bytes under way). Ten rounds are 20 wide products and about 60 other instructions for eight elements, issue slots 59 % busy; 32 bits an element would
// double that and no longer hide behind the loads.
#include "common.cuh"

namespace ve {

struct DropoutParams {
  const void *x, *res;          // [rows, cols], pitches in elements; res may be null
  long ldx, ldr;
  void* y;                      // [rows, cols], contiguous
  int rows, cols;
  uint32_t groups, div_mul;     // groups of eight columns of a row; i / groups = i * div_mul >> (31 + div_shift) for i < 2^31
  int div_shift;
  uint32_t threshold;           // t * 65536 (t = 65536 never gets here)
  float scale;
  unsigned long long seed;
  const unsigned long long* seed_at;       // on the device, in place of seed
  unsigned long long row0;
  uint32_t site;
};

VE_DEVINL uint4 philox10(uint4 c, uint2 k) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const unsigned long long a = (unsigned long long)0xD2511F53u * c.x, b = (unsigned long long)0xCD9E8D57u * c.z;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k.x, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k.y, (uint32_t)a);
    k.x += 0x9E3779B9u;
    k.y += 0xBB67AE85u;
  }
  return c;
}

// Eight elements of a row; `n` of them exist.
template <typename T, bool VEC>
VE_DEVINL void load8(const T* p, int n, float* v) {
  if (VEC) {
    if (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[2 * e] = __uint_as_float(w[e] << 16); v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? (float)p[e] : 0.f;
  }
}

template <typename T, bool VEC, bool RES>
__global__ void __launch_bounds__(256) dropout_kernel(const DropoutParams p) {
  // Groups of a thread whose loads are under way at once: with a residual one (two took 160 us where one takes 153, 16384 x 5120 forward and gradient),
  // without two: half the bytes.
  constexpr int N = RES ? 1 : 2;
  grid_dep_launch();
  grid_dep_wait();
  const unsigned long long seed = p.seed_at ? *p.seed_at : p.seed;
  const uint2 key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
  const uint32_t total = (uint32_t)p.rows * p.groups, step = gridDim.x * blockDim.x;
  for (uint32_t i0 = blockIdx.x * blockDim.x + threadIdx.x; i0 < total; i0 += N * step) {
    float x[N][8], y[8];
    uint32_t r[N], g[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const uint32_t i = u ? min(i0 + u * step, total - 1) : i0;
      r[u] = (uint32_t)((unsigned long long)i * p.div_mul >> (31 + p.div_shift));
      g[u] = i - r[u] * p.groups;
      load8<T, VEC>((const T*)p.x + (size_t)r[u] * p.ldx + g[u] * 8, min(8, p.cols - (int)(g[u] * 8)), x[u]);
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (u && i0 + u * step >= total) break;
      const int c = (int)(g[u] * 8), n = min(8, p.cols - c);
      if (RES) load8<T, VEC>((const T*)p.res + (size_t)r[u] * p.ldr + c, n, y);
      const unsigned long long row = p.row0 + r[u];
      const uint4 w4 = philox10(make_uint4(g[u], (uint32_t)row, (uint32_t)(row >> 32), p.site), key);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // 16 bits against t as 32 against t * 65536: a high half needs no extraction
        const bool keep = (e & 1 ? w[e >> 1] : w[e >> 1] << 16) >= p.threshold;       // (a choice, not a product: what stands in a dropped place does not matter)
        if (RES) y[e] = keep ? fmaf(x[u][e], p.scale, y[e]) : y[e];
        else y[e] = keep ? x[u][e] * p.scale : 0.f;
      }
      T* dst = (T*)p.y + (size_t)r[u] * p.cols + c;
      if (VEC) {
        if (sizeof(T) == 4) {
          *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
          *(reinterpret_cast<float4*>(dst) + 1) = make_float4(y[4], y[5], y[6], y[7]);
        } else {
          uint32_t b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(y[2 * e], y[2 * e + 1]);
            b[e] = *reinterpret_cast<const uint32_t*>(&v);
          }
          *reinterpret_cast<uint4*>(dst) = make_uint4(b[0], b[1], b[2], b[3]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) dst[e] = (T)y[e];
      }
    }
  }
}

template <typename T, bool VEC>
static void launch_dropout(const DropoutParams& p, cudaStream_t st) {
  const uint32_t total = (uint32_t)p.rows * p.groups;
  const int grid = (int)((total + 255) / 256 < 148 * 8 ? (total + 255) / 256 : 148 * 8);
  if (p.res) launch_pdl(dropout_kernel<T, VEC, true>, dim3(grid), dim3(256), 0, st, p);
  else launch_pdl(dropout_kernel<T, VEC, false>, dim3(grid), dim3(256), 0, st, p);
}

template <typename T>
static int run_dropout(DropoutParams p, long rows, cudaStream_t st) {
  const bool vec = p.cols % 8 == 0 && !((uintptr_t)p.x & 15) && !((uintptr_t)p.y & 15) && p.ldx * sizeof(T) % 16 == 0 &&
                   (!p.res || (!((uintptr_t)p.res & 15) && p.ldr * sizeof(T) % 16 == 0));
  const long most = (0x7fffffffl - 2 * 148 * 8 * 256) / p.groups;       // (two steps behind the last group stay below 2^31 too)
  for (long r = 0; r < rows; r += most) {
    DropoutParams q = p;
    q.rows = (int)(rows - r < most ? rows - r : most);
    q.x = (const T*)p.x + r * p.ldx;
    if (p.res) q.res = (const T*)p.res + r * p.ldr;
    q.y = (T*)p.y + r * p.cols;
    q.row0 = p.row0 + r;
    if (vec) launch_dropout<T, true>(q, st);
    else launch_dropout<T, false>(q, st);
  }
  return (int)cudaGetLastError();
}

}  // namespace ve

using namespace ve;

extern "C" {

// x, residual (or null), y: fp32 or bf16 [rows, cols], pitches ldx / ldr, y contiguous; drops where 16 bits of the generator are below `threshold` (0..65536).
int ve_dropout(const void* x, long ldx, const void* residual, long ldr, void* y, int fp32, long rows, int cols, int threshold, float scale, long seed,
               const void* seed_at, long row0, int site, cudaStream_t st) {
  if (rows <= 0 || cols <= 0) return 0;
  if (threshold < 0 || threshold > 65536) return cudaErrorInvalidValue;
  if (threshold == 65536) {              // nothing is kept
    const size_t row = (size_t)cols * (fp32 ? 4 : 2);
    return (int)(residual ? cudaMemcpy2DAsync(y, row, residual, (size_t)ldr * (fp32 ? 4 : 2), row, rows, cudaMemcpyDeviceToDevice, st)
                          : cudaMemsetAsync(y, 0, row * rows, st));
  }
  DropoutParams p{x, residual, ldx, ldr, y, 0, cols, (uint32_t)((cols + 7l) / 8), 0, 0, (uint32_t)threshold << 16, scale, (unsigned long long)seed,
                  (const unsigned long long*)seed_at, (unsigned long long)row0, (uint32_t)site};
  while ((1ul << p.div_shift) < p.groups) ++p.div_shift;
  p.div_mul = (uint32_t)(((1ull << (31 + p.div_shift)) + p.groups - 1) / p.groups);
  return fp32 ? run_dropout<float>(p, rows, st) : run_dropout<__nv_bfloat16>(p, rows, st);
}

}  // extern "C"
