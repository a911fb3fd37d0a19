// Dropout on a residual branch from a counter-based generator:
//
//   out[e] = x[e] + (r(e) >= threshold ? y[e] * gain : 0),  gain = 1 / (1 - p)
//
// r(e) is word e % 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel
// random numbers: as easy as 1, 2, 3", 2011) at the counter (e / 4 low, e / 4
// high, offset low, offset high) under the key (seed low, seed high), e the
// element's row-major index. The keep decision depends on (seed, offset, e)
// alone, so the backward pass (the same call without x, on the gradient)
// draws it again and no mask is stored, whatever layout or launch it takes.
//
// Bound: HBM (x, y read, out written; 10 B an element for an fp32 stream and
// a bf16 branch), with the generator close behind: one Philox block serves four
// elements, ten rounds of two wide multiplies and two three-way xors. Eight
// elements a thread (two blocks, 16- and 32-byte accesses). 262,144 x 256 from
// a cold L2: 104 us forward and 84 us backward; 185 to 190 us for the two in turn,
// 88 to 90% of the measured HBM rate (the generator took 72-76% of issue slots
// before the round keys were added up on the host).
#include "common.cuh"

namespace mb {
namespace drop {

constexpr int kThreads = 256;

struct Philox {
  uint32_t w[4];
};

// The ten rounds' keys, added up on the host: they are the same for every
// element, and the kernels read them as constants.
struct Keys {
  uint32_t k[20];
};
inline Keys round_keys(uint64_t seed) {
  Keys keys;
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
  for (int i = 0; i < 10; ++i) {
    keys.k[2 * i] = k0;
    keys.k[2 * i + 1] = k1;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return keys;
}

__device__ __forceinline__ Philox philox(uint64_t block, uint64_t offset, const Keys& keys) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ keys.k[2 * i];
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ keys.k[2 * i + 1];
    c3 = (uint32_t)a;
  }
  return {{c0, c1, c2, c3}};
}

// A dropped element adds nothing, whatever y holds there (NaN included).
__device__ __forceinline__ float kept(uint32_t r, uint64_t threshold, float y, float gain) {
  return (uint64_t)r >= threshold ? y * gain : 0.f;
}

// Contiguous rows: eight consecutive elements (two Philox blocks) a thread.
template <typename TX, typename TY, typename TO>
__global__ void __launch_bounds__(kThreads) flat_kernel(const TX* __restrict__ x, const TY* __restrict__ y, int64_t n,
                                                        uint64_t threshold, float gain, const Keys keys,
                                                        uint64_t offset, TO* __restrict__ out) {
  const int64_t e = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 8;
  if (e >= n) return;
  if (e + 8 <= n) {
    float ys[8], xs[8];
    load_vec<8>(y + e, ys);
    if (x) {
      load_vec<8>(x + e, xs);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) xs[i] = 0.f;
    }
    const Philox a = philox(e >> 2, offset, keys), b = philox((e >> 2) + 1, offset, keys);
#pragma unroll
    for (int i = 0; i < 8; ++i) xs[i] += kept(i < 4 ? a.w[i] : b.w[i - 4], threshold, ys[i], gain);
    store_vec<8>(out + e, xs);
  } else {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const Philox a = philox((e >> 2) + half, offset, keys);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t at = e + half * 4 + i;
        if (at < n) out[at] = from_f<TO>((x ? to_f(x[at]) : 0.f) + kept(a.w[i], threshold, to_f(y[at]), gain));
      }
    }
  }
}

// Strided or unaligned rows: four consecutive elements (one block) a thread.
template <typename TX, typename TY, typename TO>
__global__ void __launch_bounds__(kThreads) rows_kernel(const TX* __restrict__ x, int64_t ldx,
                                                        const TY* __restrict__ y, int64_t ldy, int64_t n,
                                                        int64_t width, uint64_t threshold, float gain, const Keys keys,
                                                        uint64_t offset, TO* __restrict__ out, int64_t ldo) {
  const int64_t block = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (block * 4 >= n) return;
  const Philox r = philox(block, offset, keys);
  int64_t row = block * 4 / width, col = block * 4 - row * width;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (block * 4 + i >= n) return;
    out[row * ldo + col] = from_f<TO>((x ? to_f(x[row * ldx + col]) : 0.f) +
                                      kept(r.w[i], threshold, to_f(y[row * ldy + col]), gain));
    if (++col == width) {
      col = 0;
      ++row;
    }
  }
}

}  // namespace drop
}  // namespace mb

using namespace mb;

extern "C" int mb_dropout_add(const void* x, int x_dtype, int64_t ldx, const void* y, int y_dtype, int64_t ldy,
                              int64_t rows, int64_t width, int64_t threshold, float gain, int64_t seed, int64_t offset,
                              void* out, int out_dtype, int64_t ldo, void* stream) {
  MB_REQUIRE(valid_dtype(y_dtype) && valid_dtype(out_dtype) && (!x || valid_dtype(x_dtype)), "dropout_add: bad dtype");
  MB_REQUIRE(rows >= 0 && width >= 0, "dropout_add: negative size");
  MB_REQUIRE(threshold >= 0 && threshold <= (int64_t(1) << 32), "dropout_add: threshold must be in [0, 2^32]");
  if (rows == 0 || width == 0) return MB_OK;
  MB_REQUIRE(y && out, "dropout_add: null pointer");
  MB_REQUIRE((rows == 1) || (ldy >= width && ldo >= width && (!x || ldx >= width)),
             "dropout_add: a row stride is below the width");
  MB_REQUIRE(rows <= (int64_t(1) << 40) / width, "dropout_add: too many elements");
  const int64_t n = rows * width;
  const drop::Keys keys = drop::round_keys((uint64_t)seed);
  if (!x) x_dtype = out_dtype;
  const bool flat = (rows == 1 || (ldy == width && ldo == width && (!x || ldx == width))) && aligned(y, 16) &&
                    aligned(out, 16) && aligned(x, 16);
  cudaStream_t s = as_stream(stream);
  MB_DISPATCH_T(x_dtype, TX, [&] {
    MB_DISPATCH_T(y_dtype, TY, [&] {
      MB_DISPATCH_T(out_dtype, TO, [&] {
        if (flat)
          drop::flat_kernel<<<(unsigned)cdiv(n, 8 * drop::kThreads), drop::kThreads, 0, s>>>(
              (const TX*)x, (const TY*)y, n, (uint64_t)threshold, gain, keys, (uint64_t)offset, (TO*)out);
        else
          drop::rows_kernel<<<(unsigned)cdiv(cdiv(n, 4), drop::kThreads), drop::kThreads, 0, s>>>(
              (const TX*)x, ldx, (const TY*)y, ldy, n, width, (uint64_t)threshold, gain, keys,
              (uint64_t)offset, (TO*)out, ldo);
      });
    });
  });
  return launch_status("dropout_add");
}
