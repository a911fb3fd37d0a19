// Bucketed relative-bias attention on the 5th-generation tensor cores (see
// bucket_attention.cuh for the formulas): bf16 q, k, v with head sizes 32, 64
// and 128, rows on 16 bytes. Products in TMEM (fp32), softmax, statistics and bias
// sums in fp32; the probabilities and dS are rounded to bf16 as the second
// products' operands.
//
// A pair's bias: coordinates are kept relative to the query tile's first one,
// both components in one word (16 bits each, keys saturated far outside the
// map's reach), so an offset is one subtraction, its clamp two 16-bit SIMD
// instructions, its map address one two-way dot product, and its bias one
// shared load from the head's bias spread over the map. Tiles whose queries
// spread beyond +-4095, and maps too wide for the dot product's 8-bit
// factors, take saturating offsets pair by pair instead.
#include <algorithm>
#include <type_traits>

#include "bucket_attention.cuh"
#include "sm100.cuh"

namespace mb {
namespace bucket {
namespace tc {

using namespace sm100;

constexpr int kOff = 16384;    // added to a key's components: no borrow between the halves
constexpr int kNear = 4095;    // queries' reach from the tile's first one
constexpr int kFar = 12287;    // keys' saturation: kFar - kNear passes every map radius
constexpr float kNone = -1e30f;  // running maximum before the first key

__device__ __forceinline__ int saturate(int c, int base) {
  return min(max(sub_sat(c, base), -kFar), kFar);
}
// A packed half-word pair is (first component high, second low).
__device__ __forceinline__ int pack_key(int2 c, int2 base) {
  return ((saturate(c.x, base.x) + kOff) << 16) + (saturate(c.y, base.y) + kOff);
}
__device__ __forceinline__ bool near_base(int2 c, int2 base) {
  const int x = sub_sat(c.x, base.x), y = sub_sat(c.y, base.y);
  return x >= -kNear && x <= kNear && y >= -kNear && y <= kNear;
}
__device__ __forceinline__ int pack_query(int2 c, int2 base) {  // near_base(c, base)
  return ((c.x - base.x) << 16) + (c.y - base.y);
}

// Shared-memory address of the map entry of packed (key - query), entries
// of BYTES bytes from `tab`.
struct MapIndex {
  unsigned lo, hi, coef, base;
};
template <int BYTES>
__device__ __forceinline__ MapIndex map_index(const Args& a, uint32_t tab) {
  MapIndex m;
  m.lo = ((unsigned)(kOff - a.rq) << 16) | (unsigned)(kOff - a.rr);
  m.hi = ((unsigned)(kOff + a.rq) << 16) | (unsigned)(kOff + a.rr);
  const unsigned span = 2 * a.rr + 1;
  m.coef = BYTES | (BYTES * span) << 8;
  m.base = tab - BYTES * ((unsigned)(kOff - a.rq) * span + (unsigned)(kOff - a.rr));
  return m;
}
__device__ __forceinline__ uint32_t entry_addr(const MapIndex& m, int key, int query) {
  const unsigned d = __vmins2(__vmaxs2((unsigned)(key - query), m.lo), m.hi);
  return __dp2a_lo(d, m.coef, m.base);
}
template <int BYTES>
__device__ __forceinline__ uint32_t entry_addr_far(const Args& a, uint32_t tab, int2 key, int2 query) {
  return tab + BYTES * (uint32_t)entry_of(a, query, key);
}
// The dot product's second factor (BYTES x the map's width) has 8 bits.
template <int BYTES>
__device__ __forceinline__ bool narrow_map(const Args& a) { return BYTES * (2 * a.rr + 1) <= 255; }

__device__ __forceinline__ float lds(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void lds2(uint32_t addr, float& x, uint32_t& y) {
  uint32_t u;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(u), "=r"(y) : "r"(addr));
  x = __uint_as_float(u);
}
__device__ __forceinline__ void sts(uint32_t addr, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Operand tiles of ROWS rows of D bf16, 8-row groups contiguous: 64-byte rows and
// swizzle at D = 32, 128-byte ones at D = 64, two blocks of those side by side
// at D = 128. Read K-major (summed over the dims, 16 of them a step) or MN-major
// (summed over the rows; the blocks' distance is the leading offset).
template <int D, int ROWS>
struct Tile {
  static_assert(D == 32 || D == 64 || D == 128, "head sizes of the tensor-core path");
  static constexpr int ROW = D == 32 ? 64 : 128;
  static constexpr int CHUNKS = D / 8;
  static constexpr int BLOCK = ROWS * 128;  // D = 128: bytes of a block
  static constexpr uint64_t DESC = ((uint64_t)(D == 128 ? BLOCK >> 4 : 1) << 16) | ((uint64_t)(8 * ROW >> 4) << 32) |
                                   ((uint64_t)1 << 46) | ((uint64_t)(D == 32 ? 4 : 2) << 61);
  static __device__ __forceinline__ int at(int r, int c) {  // byte offset of 16-byte chunk c of row r
    return D == 32 ? r * 64 + ((c ^ ((r >> 1) & 3)) << 4)
                   : (c >> 3) * BLOCK + r * 128 + (((c & 7) ^ (r & 7)) << 4);
  }
  static __device__ __forceinline__ uint64_t desc(uint32_t addr) { return (uint64_t)((addr >> 4) & 0x3FFF) | DESC; }
  static __device__ __forceinline__ uint64_t dims(uint32_t base, int step) {
    return desc(base + step / 4 * BLOCK + step % 4 * 32);
  }
  static __device__ __forceinline__ uint64_t rows(uint32_t base, int step) { return desc(base + step * 16 * ROW); }
};

constexpr uint32_t kTransA = 1u << 15, kTransB = 1u << 16;  // MN-major operands in the instruction descriptor

__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 columns of this thread's TMEM lane, without the wait.
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld_wait(float* v, int n) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  // the values are written by the loads above: keep their uses below the wait
#pragma unroll
  for (int i = 0; i < n; ++i) asm volatile("" : "+f"(v[i]));
}
// 64 columns of this thread's TMEM lane, waited for.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float* v) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
// 16 columns from each of two addresses, waited for.
__device__ __forceinline__ void tmem_ld16x2(uint32_t t0, uint32_t t1, float* v0, float* v1) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(t0), "r"(t1)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v0[i] = __uint_as_float(r[i]);
#pragma unroll
  for (int i = 0; i < 16; ++i) v1[i] = __uint_as_float(r[16 + i]);
}
// 32 columns from each of two addresses, waited for.
__device__ __forceinline__ void tmem_ld32x2(uint32_t t0, uint32_t t1, float* v0, float* v1) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(t0), "r"(t1)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v0[i] = __uint_as_float(r[i]);
#pragma unroll
  for (int i = 0; i < 32; ++i) v1[i] = __uint_as_float(r[32 + i]);
}
// 16 columns of this thread's TMEM lane, without the wait.
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
// 16 words to 16 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// 8 words to 8 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

__device__ __forceinline__ int2 coords_at(const Args& a, int64_t p, int r, int n) {
  const int32_t* c = a.coords + p * a.c_pos + 2 * (int64_t)r;
  return r < n ? make_int2(__ldg(c), __ldg(c + 1)) : make_int2(0, 0);
}

// Rows [r0, r0 + ROWS) of a (rows, D) operand by 16-byte asynchronous copies;
// rows at or past n are zero.
template <int D, int ROWS, int THREADS>
__device__ __forceinline__ void stage_async(uint32_t dst, const __nv_bfloat16* src, int64_t ld, int r0, int n) {
  using T = Tile<D, ROWS>;
  constexpr int STEP = THREADS / T::CHUNKS;  // rows a round; a multiple of 8, so the swizzle stays
  static_assert(STEP % 8 == 0, "a round must keep the swizzle");
  const int r = threadIdx.x / T::CHUNKS, c = threadIdx.x % T::CHUNKS;
  if (ROWS < STEP && r >= ROWS) return;
  const __nv_bfloat16* from = src + (int64_t)(r0 + r) * ld + c * 8;
  uint32_t to = dst + T::at(r, c);
#pragma unroll
  for (int i = 0; i < (ROWS + STEP - 1) / STEP; ++i) {
    const bool live = r0 + r + i * STEP < n;
    cp_async16_zfill(to, live ? from : src, live);
    from += STEP * ld;
    to += STEP * T::ROW;
  }
}

// The smallest and largest components of a warp's live coordinates, relative
// to the base and saturated; an offset range whose clamp is one map entry
// spares a tile the entry of each pair.
struct Box {
  int x0, x1, y0, y1;
  __device__ __forceinline__ void join(const Box& o) {
    x0 = min(x0, o.x0), x1 = max(x1, o.x1), y0 = min(y0, o.y0), y1 = max(y1, o.y1);
  }
};
__device__ __forceinline__ Box warp_box(int x, int y, bool live) {
  return {__reduce_min_sync(0xffffffffu, live ? x : kFar), __reduce_max_sync(0xffffffffu, live ? x : -kFar),
          __reduce_min_sync(0xffffffffu, live ? y : kFar), __reduce_max_sync(0xffffffffu, live ? y : -kFar)};
}
// The one map entry of every offset key - query between the boxes, or -1.
__device__ __forceinline__ int single_entry(const Args& a, const Box& key, const Box& query) {
  const int x0 = min(max(key.x0 - query.x1, -a.rq), a.rq), x1 = min(max(key.x1 - query.x0, -a.rq), a.rq);
  const int y0 = min(max(key.y0 - query.y1, -a.rr), a.rr), y1 = min(max(key.y1 - query.y0, -a.rr), a.rr);
  return x0 == x1 && y0 == y1 ? (x0 + a.rq) * (2 * a.rr + 1) + y0 + a.rr : -1;
}

// ---------------------------------------------------------------- forward --
// One CTA of 128 threads per (position, head, 128 queries). A thread owns a
// query row (its TMEM lane). Key tiles of 32 (head size 32, six CTAs per SM)
// or 64 (head size 64, four, and 128, two: what TMEM holds; against this choice
// 1,024 positions x 8 heads x 32-256 tokens take 6% more with 64-key tiles at four
// CTAs and 11% more with 32 at eight, whose 64 registers spill): S = Q K^T into
// TMEM, biased scores and exponentials in registers, P as bf16 back over S,
// O += P V with P read from TMEM. One commit covers PV(j) and S(j + 1), and
// K and V of tile j + 1 are copied while tile j's softmax runs. The running
// maximum that P and O are relative to is raised only when a tile's maximum
// passes it by 2^8 (O is then rescaled in TMEM), which the final division
// undoes exactly. Serving rounds P to bf16 once, the type that the product takes:
// 2^-9 of each term, next to the output's own 2^-9 (2.3e-3 off 64 bits in all, 1.7e-3
// for the output's rounding alone). For the backward pass (FULL) P is carried
// as the sum of two bf16 values: delta = dO . out must match sum P dP of the
// recomputed fp32 P to about 2^-18, or the bias sums, where dS cancels, keep P's
// 2^-9. O accumulates in TMEM, which truncates by 2^-24 a step of 16 keys: at 512 k
// keys the serving form's sums are off by bf16's own half step, and FULL's are
// flushed every 512 keys.
//
// Bound: issue and the latencies around it, not the tensor cores (6% active at
// head size 32, 23% at 64) nor HBM. 1,024 positions x 8 heads x 32-256 tokens,
// head size 32: 274 us, 55% of issue slots (about 14 instructions a pair, five of
// them the bias); 2 x 8 heads x 4,096 tokens, head size 64, a line: 159 us, 49% of
// issue slots and 45% of the exponential unit (tiles of one bucket take no lookup:
// 271 us without that); 2 x 8 heads x 1,024 tokens, head size 128: 36 us.
constexpr int FQ = 128, kFwdThreads = 128;
constexpr int kFlushKeys = 512;  // keys that the backward pass's `full` output accumulates in TMEM at a time

template <int D>
struct FwdPlan {
  static constexpr int FK = D == 32 ? 32 : 64;  // keys per tile
  static constexpr int CTAS = D == 32 ? 6 : D == 64 ? 4 : 2;         // per SM
  static constexpr int TMEM = D == 32 ? 64 : D == 64 ? 128 : 256;  // S: FK columns, O: D
  static constexpr int Q = 0, K = FQ * D * 2, V = K + 2 * FK * D * 2, KPK = V + 2 * FK * D * 2,
                       KXY = KPK + 2 * FK * 4, BOX = KXY + 2 * FK * 8, BAR = BOX + 8 * 16, TAB = BAR + 32;
};

template <int D, bool FULL>
__global__ void __launch_bounds__(kFwdThreads, FwdPlan<D>::CTAS) forward_kernel(const Args a) {
  using P = FwdPlan<D>;
  constexpr int FK = P::FK, kFlush = kFlushKeys / FK, BOXES = FK / 32;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  int* kpk = reinterpret_cast<int*>(smem + P::KPK);
  int2* kxy = reinterpret_cast<int2*>(smem + P::KXY);
  Box* box = reinterpret_cast<Box*>(smem + P::BOX);  // the keys' [stage][warp], the queries' [warp]
  float* tab = reinterpret_cast<float*>(smem + P::TAB);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + P::BAR);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(bar + 2);

  const int tid = threadIdx.x, warp = tid >> 5;
  const int n_tiles = (int)((a.length + FQ - 1) / FQ);
  const int tile = blockIdx.x % n_tiles, h = (blockIdx.x / n_tiles) % a.heads;
  const int64_t p = blockIdx.x / n_tiles / a.heads;
  const int kvh = h / (a.heads / a.kv_heads);
  const int nv = valid_of(a, p), q0 = tile * FQ, row = q0 + tid;
  const int64_t at = (p * a.heads + h) * a.length + row;
  __nv_bfloat16* orow = (__nv_bfloat16*)a.out + p * a.so.pos + h * a.so.head + row * a.so.row;
  if (q0 >= nv) {  // no query of this tile
    if (row < a.length) {
      const float zero[8] = {};
#pragma unroll
      for (int i = 0; i < D / 8; ++i) store_vec<8>(orow + 8 * i, zero);
      if (FULL)
#pragma unroll
        for (int i = 0; i < D / 8; ++i) store_vec<8>(a.full + at * D + 8 * i, zero);
      if (a.lse) a.lse[at] = -INFINITY;
    }
    return;
  }
  if (tid == 0) {
    mbar_init(smem_u32(bar), 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(P::TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const __nv_bfloat16* qb = (const __nv_bfloat16*)a.q + p * a.sq.pos + h * a.sq.head;
  const __nv_bfloat16* kb = (const __nv_bfloat16*)a.k + p * a.sk.pos + kvh * a.sk.head;
  const __nv_bfloat16* vb = (const __nv_bfloat16*)a.v + p * a.sv.pos + kvh * a.sv.head;
  const int2 base = coords_at(a, p, q0, nv), cq = row < nv ? coords_at(a, p, row, nv) : base;
  // tile j into stage j & 1: the copies and the coordinates' loads first, the
  // coordinates' words when they have come
  int2 ck = base;
  auto load_keys = [&](int j) {
    const int s = j & 1, k0 = j * FK;
    stage_async<D, FK, kFwdThreads>(sbase + P::K + s * FK * D * 2, kb, a.sk.row, k0, nv);
    stage_async<D, FK, kFwdThreads>(sbase + P::V + s * FK * D * 2, vb, a.sv.row, k0, nv);
    cp_async_commit();
    if (tid < FK) ck = k0 + tid < nv ? coords_at(a, p, k0 + tid, nv) : base;
  };
  auto place_keys = [&](int j) {
    const int s = j & 1;
    if (tid < FK) {
      kxy[s * FK + tid] = ck;
      kpk[s * FK + tid] = pack_key(ck, base);
      const Box b = warp_box(saturate(ck.x, base.x), saturate(ck.y, base.y), j * FK + tid < nv);
      if ((tid & 31) == 0) box[BOXES * s + warp] = b;
    }
  };
  {
    const Box b = warp_box(saturate(cq.x, base.x), saturate(cq.y, base.y), row < nv);
    if ((tid & 31) == 0) box[4 + warp] = b;
  }
  stage_async<D, FQ, kFwdThreads>(sbase + P::Q, qb, a.sq.row, q0, nv);
  load_keys(0);
  place_keys(0);
  const int n_map = (2 * a.rq + 1) * (2 * a.rr + 1);
  spread_bias<kFwdThreads>(a, h, tab + n_map, [&](int i, int, float b) { tab[i] = b; });
  const bool packed = __syncthreads_and(near_base(cq, base) && narrow_map<4>(a));
  const int qp = packed ? pack_query(cq, base) : 0;
  const MapIndex mi = map_index<4>(a, smem_u32(tab));
  cp_async_wait<0>();
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, t_o = tmem + FK;
  const uint32_t lane_s = tmem + ((uint32_t)(warp * 32) << 16), lane_o = lane_s + FK;
  const uint32_t tab_addr = smem_u32(tab);
  const int nk = (nv + FK - 1) / FK;
  auto issue_s = [&](int j) {
    const uint32_t q_s = sbase + P::Q, k_s = sbase + P::K + (j & 1) * FK * D * 2;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
      umma(tmem, Tile<D, FQ>::dims(q_s, s), Tile<D, FK>::dims(k_s, s), idesc_f16(FQ, FK), s);
  };
  if (tid == 0) {
    issue_s(0);
    umma_commit(smem_u32(bar));
  }
  const float2 scale2 = make_float2(a.scale * kLog2e, a.scale * kLog2e);
  Box queries = box[4];
  queries.join(box[5]);
  queries.join(box[6]);
  queries.join(box[7]);
  // a warp without a valid query takes part in the copies and barriers alone
  // (its rows of P, O and the sums stay what they were and are not stored)
  const bool rows_live = q0 + warp * 32 < nv;
  float m = kNone, l = 0.f, m_kept = kNone;
  bool ok = true;
  // O of the tiles since the last flush joins the row's running sum (relative to
  // the maximum m_kept of that time): the tensor cores' own accumulation
  // truncates, by 2^-24 a step of 16 keys. The sums stand in this tile's block
  // of `full` until its rows are written, four columns of every row at a time,
  // so that a warp's accesses are whole segments.
  const int n_rows = (int)min((int64_t)FQ, a.length - q0);
  float* kept = FULL ? a.full + (at - tid) * D + 4 * tid : nullptr;  // column c: + c * n_rows
  auto flush = [&](bool first) {
    const float f = first ? 0.f : ex2(m_kept - m);
    m_kept = m;
#pragma unroll
    for (int c = 0; c < D; c += 16) {
      float o[16];
      tmem_ld16_nowait(lane_o + c, o);
      tmem_ld_wait(o, 16);
      if (row < nv) {
        if (!first)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const float4 y = *reinterpret_cast<const float4*>(kept + (c + i) * n_rows);
            o[i] = fmaf(y.x, f, o[i]);
            o[i + 1] = fmaf(y.y, f, o[i + 1]);
            o[i + 2] = fmaf(y.z, f, o[i + 2]);
            o[i + 3] = fmaf(y.w, f, o[i + 3]);
          }
#pragma unroll
        for (int i = 0; i < 16; i += 4) store_vec<4>(kept + (c + i) * n_rows, o + i);
      }
    }
  };
  for (int j = 0; j < nk; ++j) {
    ok = ok && mbar_wait(smem_u32(bar), j & 1, abort);
    tc_fence_after();
    if (j + 1 < nk) load_keys(j + 1);
    const int s = j & 1, left = nv - j * FK;
    const bool fresh = FULL ? j % kFlush == 0 : j == 0;  // O starts anew with this tile
    if (rows_live) {
      float x[FK];
      if constexpr (FK == 64) tmem_ld64(lane_s, x);
      else tmem_ld32(lane_s, x);
      Box keys = box[BOXES * s];
      if (BOXES > 1) keys.join(box[BOXES * s + 1]);
      const int entry = packed ? single_entry(a, keys, queries) : -1;
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four chains
#pragma unroll
      for (int half = 0; half < FK; half += 32) {
        if (half > 0 && half >= left) break;  // no key
        auto biased = [&](int u, float b0, float b1) {
          const float2 y = fma2(make_float2(x[u], x[u + 1]), scale2, make_float2(b0, b1));
          x[u] = y.x;
          x[u + 1] = y.y;
        };
        if (entry >= 0) {  // every pair has one offset bucket
          const float b = tab[entry];
#pragma unroll
          for (int u = half; u < half + 32; u += 2) biased(u, b, b);
        } else if (packed) {
          const int4* k4p = reinterpret_cast<const int4*>(kpk + s * FK);
#pragma unroll
          for (int u = half; u < half + 32; u += 4) {
            const int4 k4 = k4p[u / 4];
            biased(u, lds(entry_addr(mi, k4.x, qp)), lds(entry_addr(mi, k4.y, qp)));
            biased(u + 2, lds(entry_addr(mi, k4.z, qp)), lds(entry_addr(mi, k4.w, qp)));
          }
        } else {
#pragma unroll
          for (int u = half; u < half + 32; u += 2)
            biased(u, lds(entry_addr_far<4>(a, tab_addr, kxy[s * FK + u], cq)),
                   lds(entry_addr_far<4>(a, tab_addr, kxy[s * FK + u + 1], cq)));
        }
        if (left < half + 32) {  // keys past the valid length
#pragma unroll
          for (int u = half; u < half + 32; ++u)
            if (u >= left) x[u] = -INFINITY;
        }
#pragma unroll
        for (int u = half; u < half + 32; ++u) mx[u % 4] = fmaxf(mx[u % 4], x[u]);
      }
      const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      if (FULL && fresh && j > 0) flush(j == kFlush);
      if (j == 0) {
        m = fmaxf(mt, kNone);
      } else if (__any_sync(0xffffffffu, mt > m + 8.f)) {
        const float to = mt > m + 8.f ? mt : m, f = ex2(m - to);
        m = to;
        l *= f;
        if (!fresh)
#pragma unroll
          for (int c = 0; c < D; c += 16) {
            float o[16];
            tmem_ld16_nowait(lane_o + c, o);
            tmem_ld_wait(o, 16);
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(o[i] * f);
            tmem_st16(lane_o + c, w);
          }
      }
      const float2 down = make_float2(-m, -m);
      float2 sum[4] = {};
#pragma unroll
      for (int half = 0; half < FK / 32; ++half) {
        uint32_t pk[16], lo[16];
        if (half == 0 || 32 * half < left) {
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            const int i = 32 * half + 2 * u;
            const float2 y = add2(make_float2(x[i], x[i + 1]), down), e = make_float2(ex2(y.x), ex2(y.y));
            sum[u % 4] = add2(sum[u % 4], e);
            pk[u] = bf16x2(e.x, e.y);
            if (FULL) {
              const float2 r = add2(e, make_float2(-__uint_as_float(pk[u] << 16),
                                                   -__uint_as_float(pk[u] & 0xffff0000u)));
              lo[u] = bf16x2(r.x, r.y);
            }
          }
        } else {
#pragma unroll
          for (int u = 0; u < 16; ++u) pk[u] = lo[u] = 0;
        }
        tmem_st16(lane_s + 16 * half, pk);
        if (FULL) tmem_st16(lane_s + FK / 2 + 16 * half, lo);
      }
      const float2 all = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
      l += all.x + all.y;
    }
    if (j + 1 < nk) place_keys(j + 1);
    tmem_st_wait();
    cp_async_wait<0>();
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && !*abort) {
      tc_fence_after();
      const uint32_t v_s = sbase + P::V + s * FK * D * 2;
#pragma unroll
      for (int t = 0; t < FK / 16; ++t)
        umma_ts(t_o, tmem + 8 * t, Tile<D, FK>::rows(v_s, t), idesc_f16(FQ, D) | kTransB,
                !fresh || t > 0);
      if (FULL)
#pragma unroll
        for (int t = 0; t < FK / 16; ++t)
          umma_ts(t_o, tmem + FK / 2 + 8 * t, Tile<D, FK>::rows(v_s, t), idesc_f16(FQ, D) | kTransB, 1);
      if (j + 1 < nk) issue_s(j + 1);
      umma_commit(smem_u32(bar));
    }
  }
  ok = ok && mbar_wait(smem_u32(bar), nk & 1, abort);
  tc_fence_after();
  const bool live = ok && row < nv && !(l == 0.f);
  const float inv = live ? 1.f / l : 0.f, f_kept = FULL && nk > kFlush ? ex2(m_kept - m) : 0.f;
  float o[D];
#pragma unroll
  for (int c = 0; c < D; c += 32) tmem_ld32_nowait(lane_o + c, o + c);
  tmem_ld_wait(o, D);
  if (FULL && nk > kFlush) {
    if (row < nv)
#pragma unroll
      for (int i = 0; i < D; i += 4) {
        const float4 y = *reinterpret_cast<const float4*>(kept + i * n_rows);
        o[i] = fmaf(y.x, f_kept, o[i]);
        o[i + 1] = fmaf(y.y, f_kept, o[i + 1]);
        o[i + 2] = fmaf(y.z, f_kept, o[i + 2]);
        o[i + 3] = fmaf(y.w, f_kept, o[i + 3]);
      }
    __syncthreads();  // the block's sums are read: its rows may be written
  }
#pragma unroll
  for (int i = 0; i < D; ++i) o[i] = live ? o[i] * inv : 0.f;
  if (row < a.length) {
#pragma unroll
    for (int i = 0; i < D; i += 8) store_vec<8>(orow + i, o + i);
    if (FULL)
#pragma unroll
      for (int i = 0; i < D; i += 8) store_vec<8>(a.full + at * D + i, o + i);
  }
  if (a.lse && row < a.length) a.lse[at] = live ? (m + log2f(l)) * kLn2 : -INFINITY;
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::TMEM) : "memory");
  }
}

// --------------------------------------------------------------- backward --
// A CTA takes key tiles of 128 keys of one (position, key / value head) at a
// time; a thread owns a key row (its TMEM lane), for all 64 queries of a step
// (head size 64, 128 threads) or for 32 of them (head size 32, 256 threads:
// what the smaller tiles leave of shared memory holds twice the bias sums, and
// twice the warps hide each other's latencies; head size 128 likewise). Two CTAs
// per SM, one at head size 128, whose tiles and accumulators fill it. For each query
// head of the group and each 64 queries:
//   S^T = K Q^T, dP^T = V dO^T                      (TMEM)
//   P^T = exp(s - lse) as bf16 in TMEM, dS^T = P (dP - delta) as bf16 in
//   shared memory, and dS added to the bias sums    (registers)
//   dV += P^T dO, dK += dS^T Q, dQ = dS K           (TMEM)
// dS^T is written once, rows of queries: as it is it is dK's A operand, and
// read MN-major it is dQ's. dK and dV stay in TMEM to the tile's end. P and dS are
// rounded to bf16 as operands, 2^-9 of each term like the results' own rounding;
// TMEM truncates dK's and dV's sums by 2^-24 a step of 16 queries, bf16's half step
// after 512 k queries. The bias sums take dS before its rounding.
// Bias sums: one private fp32 sum per (bucket, thread) in shared memory,
// bank = thread, so updates never conflict and every sum has a fixed order.
//
// Two ways to share the work, both fixed by the sizes and lengths alone:
// WHOLE (many positions): every CTA of one round takes a run of whole (head,
//   position) items, the runs cut where a running cost (steps, and two a tile)
//   passes the CTAs' equal shares. A run stays mostly within a head, so the
//   bias is spread and the sums are joined once per head of a run, not per
//   tile; an item's key tiles follow each other, and dQ's sum over them passes
//   through L2 to the same thread.
// else (few or long positions): one CTA per (item, key tile, part of its
//   steps); the parts of dQ (per key tile) and of dK and dV (per split) are
//   summed in their order afterwards.
//
// Bound: latency at 8 (head size 64) or 16 warps an SM, all that shared memory and
// TMEM hold. 512 positions x 8 heads x 32-256 tokens, head size 32: 370 us, 40% of
// issue slots; without the bias sums 320 us, without lookups 280 us. 16 heads on 4
// x 4,095 tokens, head size 64, a line: 560 us, 30%, then 80 us to sum dQ's parts
// (537 MB, written and read: they leave L2; summed over runs of key tiles through
// L2 instead the whole took 180 us more). 2 x 8 heads x 1,024 tokens, head size 128:
// 156 us with the delta and sums (192 TFLOP/s). One step's scores behind the last one's
// gradients changed nothing at head size 32 and cost 5% at 64.
constexpr int BQ = 64, BK = 128;

template <int D>
struct BwdPlan {
  static constexpr int THREADS = D == 64 ? 128 : 256;
  static constexpr int CTAS = D == 128 ? 1 : 2;  // per SM
  static constexpr int CH = D == 64 ? 32 : 16;   // columns a thread takes at a time
  static constexpr int T = D * 2;
  static constexpr int K = 0, V = K + BK * T, Q = V + BK * T, G = Q + 2 * BQ * T, DS = G + 2 * BQ * T,
                       QPK = DS + BK * BQ * 2, LSE = QPK + 2 * BQ * 4, DEL = LSE + 2 * BQ * 4,
                       BOX = DEL + 2 * BQ * 4, BAR = BOX + 8 * 16, TAB = BAR + 32;  // map entries (8 B, one more for dead rows), then sums
  static constexpr int TMEM = D == 128 ? 512 : 256;
};

// A position's key tiles, query steps and cost in the WHOLE sharing.
__device__ __forceinline__ int64_t cost_of(int nv, int group) {
  return 1 + (int64_t)((nv + BK - 1) / BK) * ((nv + BQ - 1) / BQ * group + 2);
}

// The first position whose items start at or past `target` of a head's cost,
// by all threads; `before` and `own` are the cost ahead of and in the thread's
// own run of positions [p0, p1).
template <int THREADS>
__device__ __forceinline__ int64_t position_at(const Args& a, int64_t target, int64_t before, int64_t own, int64_t p0,
                                               int group, int64_t* found) {
  __syncthreads();
  if (threadIdx.x == 0 && target == 0) *found = 0;
  if (before < target && target <= before + own) {
    int64_t p = p0, c = before;
    while (c < target) c += cost_of(valid_of(a, p++), group);
    *found = p;
  }
  __syncthreads();
  return *found;
}

template <int D, bool WHOLE>
__global__ void __launch_bounds__(BwdPlan<D>::THREADS, BwdPlan<D>::CTAS)
    backward_kernel(const Args a, int tile0, int n_chunk, int n_split) {
  using P = BwdPlan<D>;
  using TK = Tile<D, BK>;
  using TQ = Tile<D, BQ>;
  constexpr int THREADS = P::THREADS, CH = P::CH;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  int* qpk = reinterpret_cast<int*>(smem + P::QPK);
  Box* box = reinterpret_cast<Box*>(smem + P::BOX);  // the queries' [stage][warp], the keys' [warp]
  float* lse = reinterpret_cast<float*>(smem + P::LSE);
  float* delta = reinterpret_cast<float*>(smem + P::DEL);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + P::BAR);  // [0] scores, [1] gradients
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 2);
  volatile int* abort = reinterpret_cast<volatile int*>(bar + 3);
  const int n_map = (2 * a.rq + 1) * (2 * a.rr + 1);
  float2* tab = reinterpret_cast<float2*>(smem + P::TAB);
  float* hist = reinterpret_cast<float*>(tab + n_map + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, key = tid & (BK - 1);
  const int group = a.heads / a.kv_heads;
  const int64_t n_kv = a.n_pos * a.kv_heads * a.length * D;
  // the slot of this CTA's bias sums among those of (head, bucket)
  int64_t ctas = gridDim.x, cta = blockIdx.x;

  // ---- the CTA's work: items (head, position) in [first, last) counted
  // head-major, or one key tile of one item and steps [it0, it1) of it
  int64_t first, last;
  int sp = 0, chunk_tile = 0, only_tile = 0;
  if (WHOLE) {
    int64_t* scratch = reinterpret_cast<int64_t*>(hist);  // one sum per warp, then a result
    const int64_t per = (a.n_pos + THREADS - 1) / THREADS;
    const int64_t p0 = min(a.n_pos, tid * per), p1 = min(a.n_pos, p0 + per);
    int64_t own = 0;
    for (int64_t p = p0; p < p1; ++p) own += cost_of(valid_of(a, p), group);
    int64_t run = own;  // inclusive scan over the threads
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += up;
    }
    if (lane == 31) scratch[warp] = run;
    __syncthreads();
    int64_t before = run - own, total = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += scratch[w];
      total += scratch[w];
    }
    const int64_t lo = total * a.kv_heads * blockIdx.x / gridDim.x;
    const int64_t hi = total * a.kv_heads * (blockIdx.x + 1) / gridDim.x;
    first = lo / total * a.n_pos + position_at<THREADS>(a, lo % total, before, own, p0, group, scratch + THREADS / 32);
    last = hi / total * a.n_pos + position_at<THREADS>(a, hi % total, before, own, p0, group, scratch + THREADS / 32);
    __syncthreads();  // the scratch is read
    if (a.dbias)
      for (int64_t i = tid; i < a.heads * a.n_buckets; i += THREADS) a.bias_part[i * ctas + cta] = 0.f;
    if (first >= last) return;
  } else {
    const int n_tiles = (int)((a.length + BK - 1) / BK);
    int i = blockIdx.x;
    if (n_split > 1) sp = i % n_split, i /= n_split;
    chunk_tile = i % n_chunk, i /= n_chunk;
    only_tile = tile0 + chunk_tile;
    const int64_t p = i / a.kv_heads;
    first = i % a.kv_heads * a.n_pos + p;
    last = first + 1;
    ctas = a.n_pos * n_tiles * n_split;
    cta = (p * n_tiles + only_tile) * n_split + sp;
  }

  if (tid == 0) {
    mbar_init(smem_u32(&bar[0]), 1);
    mbar_init(smem_u32(&bar[1]), 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(P::TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, lane_t = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  // TMEM columns. dQ goes over dP^T (D = 128: and S^T). With two threads a row
  // P^T cannot go over S^T, whose other half may still be unread, and has columns
  // of its own.
  constexpr uint32_t tmem_s = 0, tmem_dp = 64, tmem_dq = D == 128 ? 0 : 64, tmem_dv = 128,
                     tmem_dk = D == 32 ? 160 : D == 64 ? 192 : 256, tmem_p = D == 32 ? 192 : D == 64 ? tmem_s : 384;
  const uint32_t tab_addr = smem_u32(tab), none_addr = tab_addr + 8 * n_map;
  const uint32_t my_hist = smem_u32(hist) + 4 * tid;
  const float2 scale2 = make_float2(a.scale * kLog2e, a.scale * kLog2e);
  const MapIndex map = map_index<8>(a, tab_addr);
  bool ok = true;
  int head = -1;       // the query head whose bias and sums are in shared memory
  uint32_t phase = 0;  // steps done: both barriers complete once a step, the stages alternate

  // the head's sums over this CTA's threads so far, a warp per bucket
  auto join_sums = [&]() {
    __syncthreads();
    if (a.dbias && head >= 0)
      for (int b = warp; b < a.n_buckets; b += THREADS / 32) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < THREADS; i += 32) sum += hist[b * THREADS + i + lane];
        sum = warp_sum(sum);
        float* dst = a.bias_part + ((int64_t)head * a.n_buckets + b) * ctas + cta;
        if (lane == 0) *dst = WHOLE ? *dst + sum : sum;
      }
    __syncthreads();
  };

  for (int64_t item = first; item < last; ++item) {
    const int kvh = (int)(item / a.n_pos);
    const int64_t p = item - kvh * a.n_pos;
    const int nv = valid_of(a, p), nq = (nv + BQ - 1) / BQ;
    // the only token of a position has P = 1 whatever its score: no gradient of
    // the scores, where dP and delta differ by their roundings
    const bool bias_sums = a.dbias && nv > 1;
    const float score_scale = nv > 1 ? a.scale : 0.f;
    const int tile_end = WHOLE ? (nv + BK - 1) / BK : only_tile + 1;
    for (int tile = WHOLE ? 0 : only_tile; tile < tile_end; ++tile) {
      const int k0 = tile * BK, row = k0 + key, n_all = k0 < nv ? group * nq : 0;
      const int64_t at = ((p * a.kv_heads + kvh) * a.length + row) * D;
      int it0 = 0, it1 = n_all;
      if (!WHOLE && n_split > 1) {
        it0 = (int)((int64_t)n_all * sp / n_split);
        it1 = (int)((int64_t)n_all * (sp + 1) / n_split);
      }
      // dk and dv values of the row's columns [c, c + 32): the result, or this split's part
      auto store_kv = [&](int which, int c, const float* o) {
        if (row >= a.length) return;
        if (!WHOLE && n_split > 1) {
          float* dst = a.dkv_part + (sp * 2 + which) * n_kv + at + c;
#pragma unroll
          for (int e = 0; e < 32; e += 8) store_vec<8>(dst + e, o + e);
        } else {
          __nv_bfloat16* dst = (__nv_bfloat16*)(which ? a.dv : a.dk) + at + c;
#pragma unroll
          for (int e = 0; e < 32; e += 8) store_vec<8>(dst + e, o + e);
        }
      };
      if (!WHOLE && a.dbias) {  // query heads without a step here
        const int h0 = it1 > it0 ? it0 / nq : 0, h1 = it1 > it0 ? (it1 - 1) / nq + 1 : 0;
        for (int i = tid; i < group * a.n_buckets; i += THREADS) {
          const int g = i / a.n_buckets;
          if (g < h0 || g >= h1) a.bias_part[((int64_t)kvh * group * a.n_buckets + i) * ctas + cta] = 0.f;
        }
      }
      if (it0 == it1) {
        const float zero[32] = {};
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          store_kv(0, c, zero);
          store_kv(1, c, zero);
        }
        continue;
      }
      // offsets are taken relative to this tile's first key: queries play the
      // saturated part here, keys the near one, and every sign is turned
      const bool live = row < nv;
      const int2 base = coords_at(a, p, k0, nv), ck = live ? coords_at(a, p, row, nv) : base;
      const int h0 = kvh * group + it0 / nq;
      // the copies and the rows' loads first, the rows' words when they have come
      int2 row_c = base;
      float row_z = 0.f, row_d = 0.f;
      bool row_live = false;
      auto load_queries = [&](int s, int h, int q0) {
        stage_async<D, BQ, THREADS>(sbase + P::Q + s * BQ * P::T,
                                    (const __nv_bfloat16*)a.q + p * a.sq.pos + h * a.sq.head, a.sq.row, q0, nv);
        stage_async<D, BQ, THREADS>(sbase + P::G + s * BQ * P::T,
                                    (const __nv_bfloat16*)a.grad + p * a.sg.pos + h * a.sg.head, a.sg.row, q0, nv);
        cp_async_commit();
        if (tid < BQ) {
          const int r = q0 + tid;
          const int64_t i = (p * a.heads + h) * a.length + r;
          row_live = r < nv;
          row_c = row_live ? coords_at(a, p, r, nv) : base;
          row_z = row_live ? a.lse_in[i] : -INFINITY;
          row_d = row_live ? a.delta[i] : 0.f;
        }
      };
      auto place_queries = [&](int s) {
        if (tid < BQ) {
          const int xs = saturate(row_c.x, base.x), ys = saturate(row_c.y, base.y);
          qpk[s * BQ + tid] = ((kOff - xs) << 16) + (kOff - ys);  // plus a key's word: offset + kOff
          const Box b = warp_box(xs, ys, row_live);
          if (lane == 0) box[2 * s + warp] = b;
          // negated; a row without a key has P = 0
          lse[s * BQ + tid] = row_z == -INFINITY ? -INFINITY : -row_z * kLog2e;
          delta[s * BQ + tid] = -row_d;
        }
      };
      stage_async<D, BK, THREADS>(sbase + P::K, (const __nv_bfloat16*)a.k + p * a.sk.pos + kvh * a.sk.head, a.sk.row,
                                  k0, nv);
      stage_async<D, BK, THREADS>(sbase + P::V, (const __nv_bfloat16*)a.v + p * a.sv.pos + kvh * a.sv.head, a.sv.row,
                                  k0, nv);
      load_queries(phase & 1, h0, (it0 - (h0 - kvh * group) * nq) * BQ);
      place_queries(phase & 1);
      {
        const Box b = warp_box(saturate(ck.x, base.x), saturate(ck.y, base.y), live);
        if (lane == 0 && warp < 4) box[4 + warp] = b;
      }
      const bool packed = __syncthreads_and(near_base(ck, base) && narrow_map<8>(a));
      MapIndex mi = map;
      if (!live) {  // a row past the valid length: every pair reads the excluded entry
        mi.coef = 0;
        mi.base = none_addr;
      }
      const int kp = packed ? -pack_query(ck, base) : 0;  // entry_addr(query word, -key): off - query + key
      Box keys = box[4];
      keys.join(box[5]);
      keys.join(box[6]);
      keys.join(box[7]);
      // a warp without a valid key keeps its rows of dS zero and does no more
      // (its rows of dV and dK are not stored)
      const bool keys_live = k0 + (warp & 3) * 32 < nv;
      if (!keys_live)
#pragma unroll
        for (int u = 0; u < BQ / 8; ++u)
          *reinterpret_cast<uint4*>(smem + P::DS + swz(key, u)) = make_uint4(0, 0, 0, 0);
      int h = h0, q0 = (it0 - (h0 - kvh * group) * nq) * BQ;
      for (int it = it0; it < it1; ++it) {
        const int s = phase & 1;
        if (h != head) {  // its bias, and its sums from zero
          if (head >= 0) join_sums();
          head = h;
          spread_bias<THREADS>(a, h, hist, [&](int i, int b, float x) {
            tab[i] = make_float2(x, __uint_as_float((uint32_t)max(b, 0) * (THREADS * 4)));
          });
          __syncthreads();  // the bias column is read
          if (tid == 0) tab[n_map] = make_float2(-INFINITY, 0.f);
          for (int i = 0; i < a.n_buckets; ++i) hist[i * THREADS + tid] = 0.f;
        }
        cp_async_wait<0>();
        fence_proxy_async();
        tc_fence_before();
        __syncthreads();  // this stage's operands and rows are written
        tc_fence_after();
        const uint32_t q_s = sbase + P::Q + s * BQ * P::T, g_s = sbase + P::G + s * BQ * P::T;
        if (tid == 0 && !*abort) {
#pragma unroll
          for (int t = 0; t < D / 16; ++t)
            umma(tmem + tmem_s, TK::dims(sbase + P::K, t), TQ::dims(q_s, t), idesc_f16(BK, BQ), t);
#pragma unroll
          for (int t = 0; t < D / 16; ++t)
            umma(tmem + tmem_dp, TK::dims(sbase + P::V, t), TQ::dims(g_s, t), idesc_f16(BK, BQ), t);
          umma_commit(smem_u32(&bar[0]));
        }
        int h_next = h, q_next = q0 + BQ;
        if (q_next >= nv) h_next = h + 1, q_next = 0;
        if (it + 1 < it1) load_queries(s ^ 1, h_next, q_next);  // the other stage's products are done
        ok = ok && mbar_wait(smem_u32(&bar[0]), s, abort);
        tc_fence_after();
        Box queries = box[2 * s];
        queries.join(box[2 * s + 1]);
        const int entry = packed ? single_entry(a, keys, queries) : -1;
        float one_b = 0.f, one_sum = 0.f;
        uint32_t one_at = 0;
        if (entry >= 0) lds2(live ? tab_addr + 8 * entry : none_addr, one_b, one_at);
        const int c_begin = (tid / BK) * (BQ * BK / THREADS), c_end = c_begin + BQ * BK / THREADS;
        // columns [c0, c0 + CH); ONE: every pair of the step has one map entry
        auto columns = [&](auto one, int c0) {
          constexpr bool ONE = decltype(one)::value;
          float x[CH], dp[CH];
          uint32_t where[CH];
          if (!ONE) {
            if (packed || !live) {
              const int4* q4p = reinterpret_cast<const int4*>(qpk + s * BQ + c0);
#pragma unroll
              for (int u = 0; u < CH; u += 4) {
                const int4 q4 = q4p[u / 4];
                where[u] = entry_addr(mi, q4.x, kp);
                where[u + 1] = entry_addr(mi, q4.y, kp);
                where[u + 2] = entry_addr(mi, q4.z, kp);
                where[u + 3] = entry_addr(mi, q4.w, kp);
              }
            } else {
#pragma unroll
              for (int u = 0; u < CH; ++u)
                where[u] = entry_addr_far<8>(a, tab_addr, ck,
                                             q0 + c0 + u < nv ? coords_at(a, p, q0 + c0 + u, nv) : base);
            }
            __syncwarp();
          }
          if constexpr (CH == 16) tmem_ld16x2(lane_t + tmem_s + c0, lane_t + tmem_dp + c0, x, dp);
          else tmem_ld32x2(lane_t + tmem_s + c0, lane_t + tmem_dp + c0, x, dp);
          uint32_t pk[CH / 2], dk[CH / 2];
          float2 sum[2] = {};
          const float4* z4 = reinterpret_cast<const float4*>(lse + s * BQ + c0);
          const float4* d4 = reinterpret_cast<const float4*>(delta + s * BQ + c0);
          auto pair = [&](int u, float z0, float z1, float dl0, float dl1) {
            float b0 = one_b, b1 = one_b;
            if (!ONE) {
              lds2(where[u], b0, where[u]);
              lds2(where[u + 1], b1, where[u + 1]);
            }
            // z and delta are stored negated. Packed pairs where registers are
            // plenty; at 128 of them their alignment costs more than it spares
            // (460 against 407 us for 512 positions of 8 heads and 256 tokens).
            float2 e, g;
            if constexpr (CH == 32) {
              const float2 y = add2(fma2(make_float2(x[u], x[u + 1]), scale2, make_float2(b0, b1)),
                                    make_float2(z0, z1));
              e = make_float2(ex2(y.x), ex2(y.y));
              g = mul2(e, add2(make_float2(dp[u], dp[u + 1]), make_float2(dl0, dl1)));
            } else {
              e = make_float2(ex2(fmaf(x[u], scale2.x, b0) + z0), ex2(fmaf(x[u + 1], scale2.x, b1) + z1));
              g = make_float2(e.x * (dp[u] + dl0), e.y * (dp[u + 1] + dl1));
            }
            pk[u / 2] = bf16x2(e.x, e.y);
            dk[u / 2] = bf16x2(g.x, g.y);
            if (ONE) {
              sum[u / 2 % 2] = add2(sum[u / 2 % 2], g);
            } else {
              dp[u] = g.x;
              dp[u + 1] = g.y;
            }
          };
#pragma unroll
          for (int u = 0; u < CH; u += 4) {
            const float4 z = z4[u / 4], dl = d4[u / 4];
            pair(u, z.x, z.y, dl.x, dl.y);
            pair(u + 2, z.z, z.w, dl.z, dl.w);
          }
          if (CH == 16) tmem_st8(lane_t + tmem_p + c0 / 2, pk);
          else tmem_st16(lane_t + tmem_p + c0 / 2, pk);
#pragma unroll
          for (int u = 0; u < CH / 8; ++u)
            *reinterpret_cast<uint4*>(smem + P::DS + swz(key, c0 / 8 + u)) =
                make_uint4(dk[4 * u], dk[4 * u + 1], dk[4 * u + 2], dk[4 * u + 3]);
          if (ONE) {
            const float2 all = add2(sum[0], sum[1]);
            one_sum += all.x + all.y;
          } else if (bias_sums) {
#pragma unroll
            for (int u = 0; u < CH; ++u) sts(my_hist + where[u], lds(my_hist + where[u]) + dp[u]);
          }
        };
#pragma unroll 1
        for (int c0 = c_begin; keys_live && c0 < c_end; c0 += CH) {
          if (q0 + c0 >= nv) {  // no query: P and dS zero
            const uint32_t zero[16] = {};
            if (CH == 16) tmem_st8(lane_t + tmem_p + c0 / 2, zero);
            else tmem_st16(lane_t + tmem_p + c0 / 2, zero);
#pragma unroll
            for (int u = 0; u < CH / 8; ++u)
              *reinterpret_cast<uint4*>(smem + P::DS + swz(key, c0 / 8 + u)) = make_uint4(0, 0, 0, 0);
          } else if (entry >= 0) {
            columns(std::true_type{}, c0);
          } else {
            columns(std::false_type{}, c0);
          }
        }
        if (bias_sums && entry >= 0) sts(my_hist + one_at, lds(my_hist + one_at) + one_sum);
        if (it + 1 < it1) place_queries(s ^ 1);
        tmem_st_wait();
        fence_proxy_async();
        tc_fence_before();
        __syncthreads();
        if (tid == 0 && !*abort) {
          tc_fence_after();
#pragma unroll
          for (int t = 0; t < BQ / 16; ++t)
            umma_ts(tmem + tmem_dv, tmem + tmem_p + 8 * t, TQ::rows(g_s, t), idesc_f16(BK, D) | kTransB,
                    it > it0 || t > 0);
#pragma unroll
          for (int t = 0; t < BQ / 16; ++t)
            umma(tmem + tmem_dk, smem_desc(sbase + P::DS + t * 32), TQ::rows(q_s, t),
                 idesc_f16(BK, D) | kTransB, it > it0 || t > 0);
#pragma unroll
          for (int t = 0; t < BK / 16; ++t)
            umma(tmem + tmem_dq, smem_desc(sbase + P::DS + t * 16 * 128), TK::rows(sbase + P::K, t),
                 idesc_f16(BQ, D) | kTransA | kTransB, t);
          umma_commit(smem_u32(&bar[1]));
        }
        // dQ: a 64-row accumulator keeps 16 rows in lanes 0-15 of each
        // quadrant; two threads a row take half of its columns each
        const int r = q0 + (warp & 3) * 16 + lane;
        const bool mine = lane < 16 && r < a.length;
        const int64_t qi = ((p * a.heads + h) * a.length + r) * D;
        constexpr int QC = D * BK / THREADS;  // columns of a thread
        const int qc = tid / BK * QC;
        const bool more = WHOLE && tile + 1 < tile_end;  // key tiles to come: the sum stays fp32
        float acc[QC];
        if (WHOLE && tile > 0 && mine) {
#pragma unroll
          for (int e = 0; e < QC; e += 4) {
            const float4 y = *reinterpret_cast<const float4*>(a.dq_part + qi + qc + e);
            acc[e] = y.x, acc[e + 1] = y.y, acc[e + 2] = y.z, acc[e + 3] = y.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < QC; ++e) acc[e] = 0.f;
        }
        ok = ok && mbar_wait(smem_u32(&bar[1]), s, abort);
        tc_fence_after();
#pragma unroll
        for (int i0 = 0; i0 < QC; i0 += 16) {
          float o[16];
          tmem_ld16_nowait(lane_t + tmem_dq + qc + i0, o);
          tmem_ld_wait(o, 16);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = ok ? fmaf(o[e], score_scale, acc[i0 + e]) : 0.f;
          if (mine) {
            float* part = WHOLE ? (more ? a.dq_part + qi : nullptr)
                                : (a.dq_part ? a.dq_part + chunk_tile * (a.n_pos * a.heads * a.length * D) + qi
                                             : nullptr);
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
              if (part) store_vec<8>(part + qc + i0 + e, o + e);
              else store_vec<8>((__nv_bfloat16*)a.dq + qi + qc + i0 + e, o + e);
            }
          }
        }
        tc_fence_before();
        ++phase;
        h = h_next;
        q0 = q_next;
      }
      tc_fence_after();
#pragma unroll
      for (int which = 0; which < 2; ++which) {  // dk, dv; one each where a row has two threads
        if (THREADS > BK && tid / BK != which) continue;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          float o[32];
          tmem_ld32(lane_t + (which ? tmem_dv : tmem_dk) + c, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = ok && live ? (which ? o[e] : o[e] * score_scale) : 0.f;
          store_kv(which, c, o);
        }
      }
      tc_fence_before();
    }
    // rows past the tiles and steps, where no sum over parts writes them
    const float zero[8] = {};
    const int64_t n = a.length * D;
    if (WHOLE) {
      const int64_t kv_at = (p * a.kv_heads + kvh) * n;
      for (int64_t e = (int64_t)tile_end * BK * D + tid * 8; e < n; e += THREADS * 8) {
        store_vec<8>((__nv_bfloat16*)a.dk + kv_at + e, zero);
        store_vec<8>((__nv_bfloat16*)a.dv + kv_at + e, zero);
      }
    }
    if (WHOLE || (!a.dq_part && sp == 0))
      for (int h = kvh * group; h < (kvh + 1) * group; ++h)
        for (int64_t e = (int64_t)nq * BQ * D + tid * 8; e < n; e += THREADS * 8)
          store_vec<8>((__nv_bfloat16*)a.dq + (p * a.heads + h) * n + e, zero);
  }
  join_sums();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::TMEM) : "memory");
  }
}

// delta_i = dO_i . out_i (out before its rounding): D / 8 lanes a row.
template <int D>
__global__ void __launch_bounds__(256) delta_kernel(const Args a) {
  constexpr int G = D / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, at = i / G;
  const int c = (int)(i % G) * 8;
  float s = 0.f;
  if (at < a.n_pos * a.heads * a.length && a.lse_in[at] != -INFINITY) {
    const int64_t row = at % a.length, h = at / a.length % a.heads, p = at / a.length / a.heads;
    float g[8], o[8];
    load_vec<8>((const __nv_bfloat16*)a.grad + p * a.sg.pos + h * a.sg.head + row * a.sg.row + c, g);
    if (a.full) load_vec<8>(a.full + at * D + c, o);
    else load_vec<8>((const __nv_bfloat16*)a.out + p * a.so.pos + h * a.so.head + row * a.so.row + c, o);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(g[e], o[e], s);
  }
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (c == 0 && at < a.n_pos * a.heads * a.length) a.delta[at] = s;
}

// dq = the sum of its key tiles' parts in their order (and of the earlier
// chunks' sum, kept in fp32), eight elements a thread; the parts of tiles past
// the valid length are not written and not read.
template <int D>
__global__ void __launch_bounds__(256) dq_sum_kernel(const Args a, int tile0, int n_chunk, float* acc, bool last) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8, n = a.n_pos * a.heads * a.length * D;
  if (e >= n) return;
  const int64_t row = e / D % a.length, p = e / D / a.length / a.heads;
  const int nv = valid_of(a, p);
  float s[8] = {};
  if (row < nv) {
    if (tile0 > 0) load_vec<8>(acc + e, s);
    const int tiles = min(n_chunk, (nv + BK - 1) / BK - tile0);
    for (int t = 0; t < tiles; ++t) {
      float x[8];
      load_vec<8>(a.dq_part + t * n + e, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += x[i];
    }
  }
  if (last) store_vec<8>((__nv_bfloat16*)a.dq + e, s);
  else store_vec<8>(acc + e, s);
}

// dk and dv as the sums of their splits' parts, in order; rows past the valid
// length, whose parts are not all written, read zero.
template <int D>
__global__ void __launch_bounds__(256) dkv_sum_kernel(const Args a, int n_split) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8, n = a.n_pos * a.kv_heads * a.length * D;
  if (e >= 2 * n) return;
  const bool second = e >= n;
  const int64_t i = second ? e - n : e, row = i / D % a.length, p = i / D / a.length / a.kv_heads;
  float s[8] = {};
  if (row < valid_of(a, p)) {
    for (int t = 0; t < n_split; ++t) {
      float x[8];
      load_vec<8>(a.dkv_part + 2 * t * n + e, x);
#pragma unroll
      for (int u = 0; u < 8; ++u) s[u] += x[u];
    }
  }
  store_vec<8>((__nv_bfloat16*)(second ? a.dv : a.dk) + i, s);
}

template <int D>
size_t backward_smem(const Args& a) {
  return BwdPlan<D>::TAB + 8 * ((size_t)(2 * a.rq + 1) * (2 * a.rr + 1) + 1) +
         (size_t)a.n_buckets * BwdPlan<D>::THREADS * 4;
}

template <int D>
int launch_forward(const Args& a, cudaStream_t s) {
  const size_t smem = FwdPlan<D>::TAB + 4 * ((size_t)(2 * a.rq + 1) * (2 * a.rr + 1) + a.n_buckets);
  auto kern = a.full ? forward_kernel<D, true> : forward_kernel<D, false>;
  if (int rc = configure(kern, smem, "bucket_attention")) return rc;
  kern<<<(unsigned)(a.n_pos * a.heads * cdiv(a.length, FQ)), kFwdThreads, smem, s>>>(a);
  return launch_status("bucket_attention");
}

template <int D>
int launch_backward(const Args& args, const BackwardPlan& plan, cudaStream_t s) {
  Args a = args;
  const int64_t tiles = cdiv(a.length, BK), n = a.n_pos * a.heads * a.length * D;
  const size_t smem = backward_smem<D>(a);
  delta_kernel<D><<<(unsigned)cdiv(n / 8, 256), 256, 0, s>>>(a);
  if (plan.whole) {
    auto kern = backward_kernel<D, true>;
    if (int rc = configure(kern, smem, "bucket_attention_backward")) return rc;
    kern<<<(unsigned)plan.ctas, BwdPlan<D>::THREADS, smem, s>>>(a, 0, 1, 1);
    return launch_status("bucket_attention_backward");
  }
  auto kern = backward_kernel<D, false>;
  if (int rc = configure(kern, smem, "bucket_attention_backward")) return rc;
  float* acc = a.dq_part;  // the chunks' running sum, then a chunk's parts
  if (tiles == 1) a.dq_part = nullptr;
  else if (tiles > plan.chunk) a.dq_part += n;
  for (int64_t t0 = 0; t0 < tiles; t0 += plan.chunk) {
    const int chunk = (int)std::min(tiles - t0, plan.chunk);
    kern<<<(unsigned)(a.n_pos * a.kv_heads * chunk * plan.split), BwdPlan<D>::THREADS, smem, s>>>(
        a, (int)t0, chunk, (int)plan.split);
    if (tiles > 1)
      dq_sum_kernel<D><<<(unsigned)cdiv(n, 8 * 256), 256, 0, s>>>(a, (int)t0, chunk, acc, t0 + chunk == tiles);
  }
  if (plan.split > 1)
    dkv_sum_kernel<D><<<(unsigned)cdiv(2 * a.n_pos * a.kv_heads * a.length * D, 8 * 256), 256, 0, s>>>(
        a, (int)plan.split);
  return launch_status("bucket_attention_backward");
}

}  // namespace tc

inline bool rows_aligned(const void* p, const Strides& s) {
  return aligned(p, 16) && s.pos % 8 == 0 && s.head % 8 == 0 && s.row % 8 == 0;
}

// bf16 tensors of head size 32, 64 or 128 whose rows are on 16 bytes; gradients of
// head size 128 with more bias sums than its tiles leave room for (about 70
// buckets) stay on the CUDA cores.
bool tc_serves(const Args& a, int dtype) {
  return dtype == MB_BF16 && (a.dim == 32 || a.dim == 64 ||
                              (a.dim == 128 && (!a.grad || tc::backward_smem<128>(a) <= 232448))) &&
         rows_aligned(a.q, a.sq) && rows_aligned(a.k, a.sk) && rows_aligned(a.v, a.sv) && rows_aligned(a.out, a.so) &&
         (!a.grad || rows_aligned(a.grad, a.sg)) && aligned(a.full, 16) && aligned(a.dq, 16) && aligned(a.dk, 16) &&
         aligned(a.dv, 16);
}

int tc_forward(const Args& a, cudaStream_t s) {
  return a.dim == 32   ? tc::launch_forward<32>(a, s)
         : a.dim == 64 ? tc::launch_forward<64>(a, s)
                       : tc::launch_forward<128>(a, s);
}

int tc_backward(const Args& a, const BackwardPlan& plan, cudaStream_t s) {
  return a.dim == 32   ? tc::launch_backward<32>(a, plan, s)
         : a.dim == 64 ? tc::launch_backward<64>(a, plan, s)
                       : tc::launch_backward<128>(a, plan, s);
}

std::atomic<int64_t> part_limit{0};

// Whole items where every CTA of one round (two per SM) has two of them or
// more. Else a launch takes as many key tiles as 2 GiB of dQ parts hold, but
// four (each launch fills the GPU, and the running sum passes through memory
// once for four parts) as long as those and the running sum stay within 16 GiB;
// beyond that fewer, one at least. 147 positions x 16 heads on 4 x 4,096 x 128,
// a part of 4.6 GiB: four tiles 173 ms and 23.0 GiB, two (taken) 187 ms and
// 13.8 GiB, one 217 ms and 9.2 GiB, whole items 178 ms and 4.7 GiB, but 114
// against 78 ms for four where the lengths differ. A caller's limit holds
// alone. Where a launch has fewer than two rounds of CTAs, a key tile's queries
// are shared by up to 16 CTAs of four steps or more.
BackwardPlan backward_plan(int64_t n_pos, int heads, int kv_heads, int head_dim, int64_t length, int dtype) {
  BackwardPlan p = {};
  if (dtype != MB_BF16 || head_dim == 16) return p;  // the CUDA-core kernels keep no parts
  constexpr int64_t round = 2 * 148;
  p.tiles = cdiv(length, tc::BK);
  const int64_t n = std::max<int64_t>(n_pos * heads * length * head_dim, 1);
  p.whole = n_pos * kv_heads >= 2 * round;
  const int64_t limit = part_limit.load(std::memory_order_relaxed);
  const int64_t least = limit ? 1 : std::clamp<int64_t>((int64_t(1) << 32) / n - 1, 1, 4);
  p.chunk = std::min(p.tiles, std::max(least, (limit ? limit : int64_t(1) << 29) / n));
  const int64_t ctas = n_pos * kv_heads * p.chunk, steps = heads / kv_heads * cdiv(length, tc::BQ);
  p.split = 1;
  while (!p.whole && p.split < 16 && ctas * p.split < 2 * round && steps / (2 * p.split) >= 4) p.split *= 2;
  p.ctas = p.whole ? round : n_pos * p.tiles * p.split;
  p.dq_words = p.tiles <= 1 ? 0 : p.whole ? n : (p.tiles > p.chunk ? p.chunk + 1 : p.chunk) * n;
  p.dkv_words = p.split > 1 ? 2 * p.split * n_pos * kv_heads * length * head_dim : 0;
  return p;
}

}  // namespace bucket
}  // namespace mb
