// The 8-bit paged K/V cache: rows quantised into their page slots, slots read
// back, and the attention of single rows and of chunks of rows over the pages.
// The reference keeps its cache in fp32 only (kernels/attention.cu:7-127); a
// decode step of long sequences is bound by the cache's bytes, which this
// format cuts to (head_dim + 1) / (2 head_dim) of bf16's.
//
// Number format.  The K (or V) slice of one token and head, x[0 .. d), is held
// as OCP e4m3 codes c and one exponent byte b:
//   e = the least integer >= -126 with max |x| <= 448 * 2^e,  b = e + 127,
//   c_i = RNE_e4m3(x_i * 2^-e),  value_i = c_i * 2^e.
// The scale is a power of two, so x * 2^-e is exact and each element is rounded
// once, to nearest even: at most 2^-4 of its value (half a step of 3 mantissa
// bits), or 2^-10 * 2^e below the normal codes.  A slice with a NaN or an
// infinity gets b = 255 and zero codes, and reads as NaN throughout: a stored
// code is never e4m3's NaN, so a bad slice cannot reach other heads or tokens
// that share a matrix instruction with it.
//
// Page layout.  A page is page_size / 16 tiles of 16 tokens; a K tile is codes
// [kv_heads][16][d] then bytes [kv_heads][16], a V tile codes [kv_heads][d][16]
// then bytes [kv_heads][16].  Both are laid out for v_mfma_f32_16x16x32: the
// scores' A operand is 16 tokens by d (lane: one token, consecutive dims), the
// output's A operand 16 dims by tokens (lane: one dim, consecutive tokens), so
// each lane's operand bytes are consecutive in memory and go from the load
// through one conversion straight into the instruction.
#include <algorithm>
#include <cmath>

#include "common.hpp"

namespace cbis {
namespace {

typedef __bf16 bf16v8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16v2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16v8_t __attribute__((ext_vector_type(8)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

constexpr int kTile = 16;          // tokens of a cache tile
constexpr int kBlk = 64;           // tokens a wave takes at a time: four tiles
constexpr int kBadByte = 255;      // scale byte of a slice with a non-finite value
constexpr int kDecodeWaves = 8;   // of a workgroup, at most
constexpr float kLowest = -3.3e38f;  // a running maximum before any score

// ---------------------------------------------------------------------------
// Addressing.
// ---------------------------------------------------------------------------
struct Pages {
  uint8_t *k, *v;
  int num_pages, page_size;
  int tshift;  // log2 of the tiles of a page
  int kv_heads, head_dim;
  int64_t tile_bytes;
};

// Byte offset of tile t of a sequence whose page there is `page`.  Page ids are
// clamped to the pool; the offset passes 32 bits in large pools.
__device__ inline int64_t tile_offset(const Pages& c, int page, int t) {
  const unsigned id = min((unsigned)page, (unsigned)(c.num_pages - 1));
  return (((int64_t)id << c.tshift) + (t & ((1 << c.tshift) - 1))) * c.tile_bytes;
}

// The wave's number in its workgroup, as a scalar: what derives from it then stays
// in scalar registers and its branches are branches.
__device__ inline int wave_id() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// A barrier that waits for the wave's LDS accesses only: __syncthreads() would
// also wait for its global loads, which are meant to stay in flight.
__device__ inline void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ inline float pow2_of_byte(unsigned b) { return __uint_as_float(b << 23); }

// ---------------------------------------------------------------------------
// Rows in and out of their slots.
//
// A workgroup of 16 waves takes up to 16 rows of 256 (fp32) or 512 (bf16) columns
// of K and of V, a row to a wave and 16 bytes of it to a lane.  Where the rows are
// the 16 tokens of one cache tile (a prompt's rows) the V codes are turned in LDS,
// so that the tile's dims are written and read in whole 16-byte pieces; other rows
// go slot by slot.  With a wave to a row and no more, the 16 bytes of a V dim came
// from up to 8 XCDs, each writing its own part of the line back (16355 bf16 rows of
// 8 heads of 128 took 103 us).
// HBM-bound on large calls: those rows are written in 23.3 us (4.3 TB/s of reads and
// writes, a large copy's rate is 4.8), 12291 bf16 rows of 64 heads of 32 read back in
// 25.5 (6.0).  By latency on small ones, so the waves share nothing they need not,
// and the code is short: it is fetched anew by every launch (8 rows 2.8 us, 777
// scattered ones read back 5.0).  Two whole rows to a wave of 8 give fp32 rows 5-9%
// and cost bf16 ones 5%; four of them cost 16%.
// Rows of at most half or a quarter of a wave's columns go two or four to a wave
// (34812 rows of 256 bf16 columns written 20.7 -> 15.6 us, read back 16.2 -> 11.4; of
// 128 columns 18.7 -> 9.7 and 15 -> 9.9).
//
// The rows are cut into groups where the tokens are: row r follows row r - 1 if
// its slot is the next one of the same tile.  A window of 16 rows owns the runs
// that start in it (which may end up to 15 rows behind it), and takes them in
// groups of whole runs of at most 16 rows.
// ---------------------------------------------------------------------------
struct RowsArgs {
  Pages c;
  int n_rows;
  const void *k, *v;
  int64_t ldk, ldv;
  const int *page, *offset;
  int parts;  // parts of 64 lanes' columns of a row
};

template <typename T>
constexpr int kLaneCols = 16 / sizeof(T);
constexpr int kRowThreads = kTile * 64;

// Rows need no more than their elements' alignment: gfx950 loads and stores
// vectors at any address.
typedef u32x4_t __attribute__((aligned(4))) u32x4_any_t;
typedef u32x4_t __attribute__((aligned(2))) u32x4_half_t;

__device__ inline bool slot_ok(const RowsArgs& a, int64_t row, int* page, int* off) {
  if (row < 0 || row >= a.n_rows) return false;
  *page = a.page[row];
  *off = a.offset[row];
  return (unsigned)*page < (unsigned)a.c.num_pages && (unsigned)*off < (unsigned)a.c.page_size;
}

// Lane i holds row window + i: its slot, and bit i whether it has one and
// whether a run starts there (rows without a slot are runs of their own).
struct RowSlots {
  int page, off;
  uint64_t starts, live;
};

__device__ inline RowSlots row_slots(const RowsArgs& a, int64_t window, int lane) {
  RowSlots r;
  int p0 = 0, o0 = 0;
  r.page = r.off = 0;
  const bool live = slot_ok(a, window + lane, &r.page, &r.off), before = slot_ok(a, window + lane - 1, &p0, &o0);
  const bool follows = live && before && r.page == p0 && r.off == o0 + 1 && (r.off & (kTile - 1)) != 0;
  r.starts = __ballot(!follows);
  r.live = __ballot(live);
  return r;
}

// The end of the group that starts at row `at` of the window: whole runs of at
// most 16 rows together, not past `end`.
__device__ inline int group_end(uint64_t starts, int at, int end) {
  const unsigned m = (unsigned)(starts >> (at + 1)) & 0xFFFFu;  // never 0: a run has at most 16 rows
  return min(at + 32 - __clz((int)m), end);
}

// Transposes 4 x 4 bytes: dword i of the result holds byte i of each w.
__device__ inline void transpose4(uint32_t* w) {
  const uint32_t t0 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), t1 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
  const uint32_t u0 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), u1 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  w[0] = __builtin_amdgcn_perm(u0, t0, 0x05040100u);
  w[1] = __builtin_amdgcn_perm(u0, t0, 0x07060302u);
  w[2] = __builtin_amdgcn_perm(u1, t1, 0x05040100u);
  w[3] = __builtin_amdgcn_perm(u1, t1, 0x07060302u);
}

__device__ inline void load_row(const float* p, float* x) {
  const u32x4_t w = __builtin_nontemporal_load((const u32x4_any_t*)p);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
}

__device__ inline void load_row(const uint16_t* p, float* x) {
  const u32x4_t w = __builtin_nontemporal_load((const u32x4_half_t*)p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16lo(w[i]);
    x[2 * i + 1] = bf16hi(w[i]);
  }
}

__device__ inline void store_row(float* p, const float* x) {
  __builtin_nontemporal_store(
      u32x4_t{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])},
      (u32x4_any_t*)p);
}

__device__ inline void store_row(uint16_t* p, const float* x) {
  __builtin_nontemporal_store(u32x4_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                      pack_bf16x2(x[6], x[7])},
                              (u32x4_half_t*)p);
}

// Maximum over aligned groups of L lanes (L = 4, 8, 16 or 32).
template <int L>
__device__ inline unsigned lanes_max(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));   // lane ^ 1
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));   // lane ^ 2
  if constexpr (L >= 8) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));   // the other 4 of 8
  if constexpr (L >= 16) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));  // of 16
  if constexpr (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((unsigned)r[0], (unsigned)r[1]);
  }
  return v;
}

// A lane's N codes of a slice held by HD / N lanes, and the slice's scale byte.
template <int HD, int N>
__device__ inline void quantise(const float* x, uint32_t* w, int* byte) {
  // max |x| by its bits: NaN above infinity above every finite value.
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  top = lanes_max<HD / N>(top);
  const bool bad = top >= 0x7F800000u;
  // max |x| = 1.m * 2^(E - 127) <= 448 * 2^e = 1.75 * 2^(8 + e): e + 127 = E - 8,
  // one more where 1.m > 1.75 (where adding 0x1FFFFF to m carries).
  const int b = max(1, (int)((top + 0x1FFFFFu) >> 23) - 8);
  const float inv = pow2_of_byte((unsigned)(254 - b));
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    int d = __builtin_amdgcn_cvt_pk_fp8_f32(x[i] * inv, x[i + 1] * inv, 0, false);
    d = __builtin_amdgcn_cvt_pk_fp8_f32(x[i + 2] * inv, x[i + 3] * inv, d, true);
    w[i / 4] = bad ? 0u : (uint32_t)d;
  }
  *byte = bad ? kBadByte : b;
}

template <int N>
__device__ inline void values(const uint32_t* w, float scale, float* x) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i / 4], false);
    const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i / 4], true);
    x[i] = lo[0] * scale;
    x[i + 1] = lo[1] * scale;
    x[i + 2] = hi[0] * scale;
    x[i + 3] = hi[1] * scale;
  }
}

// What a workgroup of the row kernels works on.  R rows to a wave (1, 2 or 4, where
// they are as narrow as that), 64 / R lanes each.
template <int HD, int N, int R>
struct RowPlace {
  int wave, lane, part, col, head, dim, at, end;
  int row;  // the lane's row of the group
  int64_t window, codes;
  bool col_ok;
  RowSlots rs;
  __device__ RowPlace(const RowsArgs& a) {
    wave = wave_id();
    lane = threadIdx.x & 63;
    window = (int64_t)(blockIdx.x / a.parts) * kTile;
    part = (int)(blockIdx.x % a.parts);
    col = (part * 64 + lane % (64 / R)) * N;
    row = wave * R + lane / (64 / R);
    col_ok = col < a.c.kv_heads * HD;
    head = col / HD;
    dim = col % HD;
    codes = (int64_t)a.c.kv_heads * HD * kTile;
    rs = row_slots(a, window, lane);
    at = rs.starts & 0xFFFF ? __ffsll((unsigned long long)rs.starts) - 1 : 64;  // 64: the window owns no row
    end = kTile + __ffsll((unsigned long long)(rs.starts >> kTile)) - 1;
  }
  // Whether rows at .. stop - 1 are a cache tile's 16 tokens.
  __device__ bool whole(int stop) const {
    return stop - at == kTile && ((rs.starts >> (at + 1)) & 0x7FFF) == 0 && (rs.live >> at & 1);
  }
  __device__ bool mine(int stop) const {
    const int i = at + (R == 1 ? wave : row);
    return i < stop && (rs.live >> i & 1);
  }
  // Offset of the tile that row at + i lies in, and its slot there.
  __device__ int64_t tile(const RowsArgs& a, int i, int* slot) const {
    const int page = __builtin_amdgcn_readlane(rs.page, at + i), off = __builtin_amdgcn_readlane(rs.off, at + i);
    return tile_at(a, page, off, slot);
  }
  // Those of the lane's own row (by all lanes of the wave).
  __device__ int64_t my_tile(const RowsArgs& a, int* slot) const {
    if constexpr (R == 1) return tile(a, wave, slot);
    else return tile_at(a, __shfl(rs.page, at + row, 64), __shfl(rs.off, at + row, 64), slot);
  }
  __device__ static int64_t tile_at(const RowsArgs& a, int page, int off, int* slot) {
    *slot = off & (kTile - 1);
    return (((int64_t)page << a.c.tshift) + (off >> 4)) * a.c.tile_bytes;
  }
};

template <typename T, int HD, int R>
__global__ __launch_bounds__(kRowThreads / R) void kv8_scatter_kernel(const RowsArgs a) {
  constexpr int N = kLaneCols<T>, NW = N / 4;
  __shared__ uint32_t turn[kTile][64 / R * NW];  // V codes of the group's rows, 4 columns to a dword
  RowPlace<HD, N, R> r(a);
  for (int stop; r.at < r.end; r.at = stop) {
    stop = group_end(r.rs.starts, r.at, r.end);
    const bool whole = r.whole(stop);
    const bool mine = r.mine(stop);
    if (R == 1 ? mine : __ballot(mine) != 0) {
      const int64_t row = r.window + r.at + (R == 1 ? r.wave : r.row);
      float xk[N] = {}, xv[N] = {};
      if (mine && r.col_ok) {
        load_row((const T*)a.k + row * a.ldk + r.col, xk);
        load_row((const T*)a.v + row * a.ldv + r.col, xv);
      }
      int slot, bk, bv;
      const int64_t tile = r.my_tile(a, &slot);
      uint32_t wk[NW], wv[NW];
      quantise<HD, N>(xk, wk, &bk);
      quantise<HD, N>(xv, wv, &bv);
      if (mine && r.col_ok) {
        uint8_t* dk = a.c.k + tile + ((int64_t)r.head * kTile + slot) * HD + r.dim;
        if constexpr (NW == 1) *(uint32_t*)dk = wk[0];
        else *(u32x2_t*)dk = u32x2_t{wk[0], wk[1]};
        if (r.dim == 0) {
          a.c.k[tile + r.codes + r.head * kTile + slot] = (uint8_t)bk;
          a.c.v[tile + r.codes + r.head * kTile + slot] = (uint8_t)bv;
        }
        if (whole) {
#pragma unroll
          for (int i = 0; i < NW; ++i) turn[R == 1 ? r.wave : r.row][r.lane % (64 / R) * NW + i] = wv[i];
        } else {
          uint8_t* dv = a.c.v + tile + (int64_t)r.col * kTile + slot;
#pragma unroll
          for (int j = 0; j < N; ++j) dv[j * kTile] = (uint8_t)(wv[j / 4] >> (8 * (j & 3)));
        }
      }
    }
    if (whole) {
      __syncthreads();
      // Thread t of the first NW waves takes columns 4 t .. 4 t + 3 of the part.
      const int col = r.part * 64 * N + 4 * (int)threadIdx.x;
      if (r.wave < NW && col < a.c.kv_heads * HD) {
        int slot;
        uint8_t* dst = a.c.v + r.tile(a, 0, &slot) + (int64_t)col * kTile;
        uint32_t w[kTile];
#pragma unroll
        for (int i = 0; i < kTile; ++i) w[i] = turn[i][threadIdx.x];
#pragma unroll
        for (int i = 0; i < kTile; i += 4) transpose4(w + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) *(u32x4_t*)(dst + j * kTile) = u32x4_t{w[j], w[4 + j], w[8 + j], w[12 + j]};
      }
      __syncthreads();
    }
  }
}

// Read back: the same groups the other way.
template <typename T, int HD, int R>
__global__ __launch_bounds__(kRowThreads / R) void kv8_gather_kernel(const RowsArgs a) {
  constexpr int N = kLaneCols<T>, NW = N / 4;
  __shared__ uint32_t turn[kTile][64 / R * NW];
  RowPlace<HD, N, R> r(a);
  for (int stop; r.at < r.end; r.at = stop) {
    stop = group_end(r.rs.starts, r.at, r.end);
    const bool whole = r.whole(stop);
    if (whole) {
      const int col = r.part * 64 * N + 4 * (int)threadIdx.x;
      if (r.wave < NW && col < a.c.kv_heads * HD) {
        int slot;
        const uint8_t* src = a.c.v + r.tile(a, 0, &slot) + (int64_t)col * kTile;
        uint32_t w[kTile];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4_t v = *(const u32x4_t*)(src + j * kTile);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[4 * i + j] = v[i];
        }
#pragma unroll
        for (int i = 0; i < kTile; i += 4) transpose4(w + i);
#pragma unroll
        for (int i = 0; i < kTile; ++i) turn[i][threadIdx.x] = w[i];
      }
      __syncthreads();
    }
    int slot;
    int64_t tile;
    if constexpr (R > 1) tile = r.my_tile(a, &slot);
    if (r.mine(stop) && r.col_ok) {
      if constexpr (R == 1) tile = r.my_tile(a, &slot);
      const uint32_t* src = (const uint32_t*)(a.c.k + tile + ((int64_t)r.head * kTile + slot) * HD + r.dim);
      uint32_t wk[NW], wv[NW];
#pragma unroll
      for (int i = 0; i < NW; ++i) wk[i] = src[i];
      if (whole) {
#pragma unroll
        for (int i = 0; i < NW; ++i) wv[i] = turn[R == 1 ? r.wave : r.row][r.lane % (64 / R) * NW + i];
      } else {
        const uint8_t* sv = a.c.v + tile + (int64_t)r.col * kTile + slot;
#pragma unroll
        for (int i = 0; i < NW; ++i)
          wv[i] = sv[4 * i * kTile] | sv[(4 * i + 1) * kTile] << 8 | sv[(4 * i + 2) * kTile] << 16 |
                  (uint32_t)sv[(4 * i + 3) * kTile] << 24;
      }
      const float sk = pow2_of_byte(a.c.k[tile + r.codes + r.head * kTile + slot]);
      const float sv = pow2_of_byte(a.c.v[tile + r.codes + r.head * kTile + slot]);
      const int64_t row = r.window + r.at + (R == 1 ? r.wave : r.row);
      float x[N];
      values<N>(wk, sk, x);
      store_row((T*)a.k + row * a.ldk + r.col, x);
      values<N>(wv, sv, x);
      store_row((T*)a.v + row * a.ldv + r.col, x);
    }
    if (whole) __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Attention.
//
// Both kernels compute S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32
// over blocks of 64 tokens (four tiles).  Row m of the scores' p-th product is
// token 4 p + m % 4 of tile m / 4, so a lane's accumulators over p = 0 .. 3 are
// the 16 tokens of tile lane / 16 for column lane % 16 -- which is the k order
// in which a lane's 16 consecutive V bytes of a dim enter the second product:
// probabilities never cross lanes.
//
// Numbers.  e4m3 codes are exact in bf16 (scores) and f16 (output).  q enters
// as QP bf16 parts: one for bf16 q; two (16 bits) for fp32 q and a bf16 result;
// three (all 24 bits) for fp32 q and an fp32 result.  The probabilities enter
// as PP f16 parts: one (11 bits) for a bf16 result, whose own rounding is 8
// bits; two (22 bits) for fp32.  f16's range is kept by two references per
// column, both raised only when a block needs it: m, with p = 2^(s - m + 8) <=
// 2^15 (s in log2 units), and E, a bound on the V scales' bytes.  Scores, sums
// and outputs are fp32.
// ---------------------------------------------------------------------------
struct AttnArgs {
  Pages c;
  int n_rows, n_heads, group;
  const int* rows;
  const void* q;
  int64_t ldq;
  int q_bf16, q_vec;
  const int* bt;
  int64_t bt_stride;
  const int *row_bt, *row_pos;
  void* out;
  int64_t ldo;
  int out_bf16, out_vec;
  int max_tok;       // tokens a block-table row covers
  float qscale;      // log2(e) / sqrt(head_dim)
  int nsplit, split_blocks;
  float *part, *lse;  // [slot][split][n_heads][head_dim] normalised outputs, [slot][split][n_heads] log2 sums
  // decode
  int nhb, tw;  // head blocks of a row, waves of a workgroup that share one
  // chunk
  const int* tiles;
  int n_tiles, ncg;  // column groups of a kv head
};

// 8 consecutive q values of a column, times scale, as QP bf16 parts.
template <int QP>
__device__ inline void load_q8(const AttnArgs& a, int64_t at, bool valid, float scale, bf16v8_t* part) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  if (valid) {
    if (a.q_bf16) {
      const uint16_t* p = (const uint16_t*)a.q + at;
      if (a.q_vec) {
        const u32x4_t w = *(const u32x4_t*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[2 * i] = bf16lo(w[i]);
          x[2 * i + 1] = bf16hi(w[i]);
        }
      } else {
        for (int i = 0; i < 8; ++i) x[i] = bf16_to_f32(p[i]);
      }
    } else {
      const float* p = (const float*)a.q + at;
      if (a.q_vec) {
        const float4 u = *(const float4*)p, v = *(const float4*)(p + 4);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
        x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
      } else {
        for (int i = 0; i < 8; ++i) x[i] = p[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= scale;
#pragma unroll
  for (int k = 0; k < QP; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __bf16 h = (__bf16)x[i];
      part[k][i] = h;
      x[i] -= (float)h;
    }
}

// First dim of the 8 that lane group g holds in k step s.
template <int HD>
__device__ inline int q_dim(int s, int g) {
  if constexpr (HD == 32) return 8 * g;
  else return 64 * (s / 2) + 16 * g + 8 * (s & 1);
}

// A lane's K bytes of one product: HD / 4 consecutive-in-16 bytes.
template <int HD>
struct KRaw {
  uint32_t w[HD / 16];
};

template <int HD>
__device__ inline KRaw<HD> load_k(const uint8_t* p) {
  KRaw<HD> r;
  if constexpr (HD == 32) {
    const u32x2_t w = __builtin_nontemporal_load((const u32x2_t*)p);
    r.w[0] = w[0];
    r.w[1] = w[1];
  } else {
#pragma unroll
    for (int h = 0; h < HD / 64; ++h) {
      const u32x4_t w = __builtin_nontemporal_load((const u32x4_t*)(p + 64 * h));
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[4 * h + i] = w[i];
    }
  }
  return r;
}

// 8 codes (two dwords) as bf16, times scale's power of two.
__device__ inline bf16v8_t codes_bf16(uint32_t lo, uint32_t hi, float scale) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16v8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ inline f16v8_t codes_f16(uint32_t lo, uint32_t hi) {
  const f16v2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
  const f16v2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  const f16v2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
  const f16v2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  return f16v8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Maximum / sum over the four lanes of a column (lanes n, n + 16, n + 32, n + 48).
__device__ inline float column_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ inline float column_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ inline int column_max(int x) {
  auto r = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false);
  x = max((int)r[0], (int)r[1]);
  r = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)x, false, false);
  return max((int)r[0], (int)r[1]);
}

__device__ inline void store_out4(const AttnArgs& a, int64_t at, const float* o) {
  if (a.out_bf16) {
    uint16_t* p = (uint16_t*)a.out + at;
    const uint2 w = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
    if (a.out_vec) {
      *(uint2*)p = w;
    } else {
      p[0] = (uint16_t)w.x; p[1] = (uint16_t)(w.x >> 16);
      p[2] = (uint16_t)w.y; p[3] = (uint16_t)(w.y >> 16);
    }
  } else {
    float* p = (float*)a.out + at;
    if (a.out_vec) {
      *(float4*)p = make_float4(o[0], o[1], o[2], o[3]);
    } else {
      for (int i = 0; i < 4; ++i) p[i] = o[i];
    }
  }
}

__device__ inline unsigned byte_of(uint32_t w, int i) { return (w >> (8 * i)) & 0xFFu; }

// Byte mask of dword d (tokens 4 d .. 4 d + 3) of a tile's first `valid` tokens.
__device__ inline uint32_t token_mask(int valid, int d) {
  const int n = min(max(valid - 4 * d, 0), 4);
  return n == 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1u;
}

__device__ inline u32x4_t keep(bool mine, u32x4_t w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = mine ? w[i] : 0u;
  return w;
}

// What single rows and tiles of few columns share: a wave's 16 columns over the
// 64-token blocks b0, b0 + step, .. below b1 of a row whose keys are 0 .. kv - 1, into
// the running maximum m, the sums l, the V scales' bound E and the outputs O.
// kCausal: the columns have last keys `pos` of their own, and every one sees the
// keys below `full`.
//
// Bound by HBM while enough bytes are in flight: a block's K and V are 32
// registers of loads each (NH * HD = 128), the next block's K is loaded as soon
// as this one's has been multiplied, V likewise, so that one of the two is
// always on its way.  Page ids are read two blocks ahead, before loads that are
// not yet wanted, since loads arrive in order and awaiting one awaits the older
// ones; they are turned into addresses only where those are used.
template <int HD, int NH, int QP, int PP, bool kCausal>
__device__ __forceinline__ void attend_keys(const AttnArgs& a, const int* bt, const bf16v8_t (&q)[HD / 32][QP], int kv, int pos,
                                   int full, int b0, int b1, int step, int kh0, int my, int my_head, bool col_ok,
                                   float& m, float& l, int& E, f32x4_t (&O)[HD / 16]) {
  constexpr int NK = HD / 32, ND = HD / 16;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int tlast = (kv - 1) >> 4;
  const int64_t codes = (int64_t)a.c.kv_heads * HD * kTile;
  // Lane offsets inside a tile; kv heads past the last one read the last.
  const int k_lane = (n & 3) * HD + (HD == 32 ? 8 : 16) * g;
  int64_t head_off[NH];
#pragma unroll
  for (int j = 0; j < NH; ++j) head_off[j] = (int64_t)min(kh0 + j, a.c.kv_heads - 1) * HD * kTile;
  const int64_t byte_off = codes + my_head * kTile;

  KRaw<HD> kr[NH][4];
  u32x4_t vr[NH][ND];
  auto load_k_block = [&](int64_t tile) {
    const uint8_t* p0 = a.c.k + tile + k_lane;
#pragma unroll
    for (int j = 0; j < NH; ++j)
#pragma unroll
      for (int p = 0; p < 4; ++p) kr[j][p] = load_k<HD>(p0 + head_off[j] + 4 * p * HD);
  };
  auto load_v_block = [&](int64_t tile) {
    const uint8_t* p0 = a.c.v + tile + n * kTile;
#pragma unroll
    for (int j = 0; j < NH; ++j)
#pragma unroll
      for (int i = 0; i < ND; ++i) vr[j][i] = __builtin_nontemporal_load((const u32x4_t*)(p0 + head_off[j] + i * kTile * kTile));
  };

  if (b0 < b1) {
    // Lane's tiles of block b, for K and for V, and the pages they are in.
    auto k_tile = [&](int b) { return min(4 * b + (n >> 2), tlast); };
    auto v_tile = [&](int b) { return min(4 * b + g, tlast); };
    const int kpage0 = bt[k_tile(b0) >> a.c.tshift], vpage0 = bt[v_tile(b0) >> a.c.tshift];
    int kpage = bt[k_tile(b0 + step) >> a.c.tshift], vpage = bt[v_tile(b0 + step) >> a.c.tshift];
    int64_t vo = tile_offset(a.c, vpage0, v_tile(b0));
    load_k_block(tile_offset(a.c, kpage0, k_tile(b0)));
    u32x4_t kb = *(const u32x4_t*)(a.c.k + vo + byte_off);  // tile g's scale bytes of the column's head
    u32x4_t vb = *(const u32x4_t*)(a.c.v + vo + byte_off);
    load_v_block(vo);
    // Behind the last block the loads go to the row's last tile again.  They are
    // not branched around: where loads may or may not have been issued, the wait
    // for older ones would be for these too.
    for (int b = b0; b < b1; b += step) {
      f32x4_t S[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) S[p] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NH; ++j) {
        const bool mine = NH == 1 || my == j;
#pragma unroll
        for (int s = 0; s < NK; ++s) {
          bf16v8_t qm[QP];
#pragma unroll
          for (int k = 0; k < QP; ++k) qm[k] = __builtin_bit_cast(bf16v8_t, keep(mine, __builtin_bit_cast(u32x4_t, q[s][k])));
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const bf16v8_t kf = codes_bf16(kr[j][p].w[2 * s], kr[j][p].w[2 * s + 1], 1.f);
#pragma unroll
            for (int k = 0; k < QP; ++k) S[p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qm[k], S[p], 0, 0, 0);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      load_k_block(tile_offset(a.c, kpage, k_tile(b + step)));
      __builtin_amdgcn_sched_barrier(0);
      const int valid = min(max(kv - (b * kBlk + g * kTile), 0), kTile);  // tokens of tile g inside the row
      const bool tail = (b + 1) * kBlk > kv, mask = kCausal ? (b + 1) * kBlk > full : tail;
      const int seen = kCausal ? pos + 1 - (b * kBlk + g * kTile) : valid;  // of them, by the column
      float top = -INFINITY;
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = S[p][i] * (pow2_of_byte(byte_of(kb[p], i)) * a.qscale);
          if (mask && 4 * p + i >= seen) x = -INFINITY;
          S[p][i] = x;
          top = fmaxf(top, x);
        }
      if (tail) {
#pragma unroll
        for (int d = 0; d < 4; ++d) vb[d] &= token_mask(valid, d);
      }
      int bmax = 0;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) bmax = max(bmax, (int)byte_of(vb[d], i));
      if (__ballot(bmax == kBadByte)) {  // a V slice of NaN: its columns' sums become NaN
        bmax = 0;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if ((int)byte_of(vb[d], i) == kBadByte) {
              if (col_ok && (!kCausal || 4 * d + i < seen)) l = NAN;
              vb[d] &= ~(0xFFu << (8 * i));
            }
            bmax = max(bmax, (int)byte_of(vb[d], i));
          }
      }
      if (__ballot(top > m + 7.f || bmax > E)) {
        const float m1 = fmaxf(m, column_max(top));
        const int E1 = max(E, column_max(bmax));
        const float r = fast_exp2(m - m1);
        l *= r;
        const float ro = ldexpf(r, E - E1);
#pragma unroll
        for (int i = 0; i < ND; ++i) O[i] *= ro;
        m = m1;
        E = E1;
      }
      // p = 2^(s - m + 8), and P' = p * 2^(byte - E) in f16 parts.
      f16v8_t P[2][PP];
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = fast_exp2(S[p][i] - (m - 8.f));
          l += e;
          float x = ldexpf(e, (int)byte_of(vb[p], i) - E);
#pragma unroll
          for (int k = 0; k < PP; ++k) {
            const _Float16 h = (_Float16)x;
            P[p / 2][k][4 * (p & 1) + i] = h;
            x -= (float)h;
          }
        }
      if (tail) {  // a slot past the row may hold anything
        const uint32_t vm[4] = {token_mask(valid, 0), token_mask(valid, 1), token_mask(valid, 2), token_mask(valid, 3)};
#pragma unroll
        for (int j = 0; j < NH; ++j)
#pragma unroll
          for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int d = 0; d < 4; ++d) vr[j][i][d] &= vm[d];
      }
#pragma unroll
      for (int j = 0; j < NH; ++j) {
        const bool mine = NH == 1 || my == j;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          f16v8_t pm[PP];
#pragma unroll
          for (int k = 0; k < PP; ++k) pm[k] = __builtin_bit_cast(f16v8_t, keep(mine, __builtin_bit_cast(u32x4_t, P[half][k])));
#pragma unroll
          for (int i = 0; i < ND; ++i) {
            const f16v8_t vf = codes_f16(vr[j][i][2 * half], vr[j][i][2 * half + 1]);
#pragma unroll
            for (int k = 0; k < PP; ++k) O[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pm[k], O[i], 0, 0, 0);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      vo = tile_offset(a.c, vpage, v_tile(b + step));
      kb = *(const u32x4_t*)(a.c.k + vo + byte_off);
      vb = *(const u32x4_t*)(a.c.v + vo + byte_off);
      kpage = bt[k_tile(b + 2 * step) >> a.c.tshift];
      vpage = bt[v_tile(b + 2 * step) >> a.c.tshift];
      __builtin_amdgcn_sched_barrier(0);
      load_v_block(vo);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// Single rows.  A workgroup owns (row, NH kv heads, split); its waves take the
// split's 64-token blocks in turn.  The 16 columns of the products are the query
// heads: with q zero outside a kv head's own columns the scores of the NH kv
// heads accumulate into the same four registers per product, each head in its
// column, so one softmax serves them all; the output does the same with P.
//
// 192 rows of 256..4096, 64 heads of 32: 264 us, 6.7 TB/s (a read-only kernel reaches
// 7.1); 16 rows of 32768: 328 and 5 of joining.  61 rows of 500..16384, 8 K/V heads
// of 128: 185 us, 5.7 TB/s, 6.6% more than its bytes fetched: 8 heads' scale bytes
// share a line that as many XCDs read.  (All heads of a row on one XCD gives 2.5%,
// but leaves XCDs idle where rows are few or unsorted.)  The non-temporal loads are
// worth 12% at 32 dims (304 us without), 3% at 128.
template <int HD, int NH, int QP, int PP>
__global__ __launch_bounds__(kDecodeWaves * 64) void kv8_decode_kernel(const AttnArgs a) {
  constexpr int NK = HD / 32, ND = HD / 16;
  constexpr int kPitch = HD + 4;
  extern __shared__ float o_sh[];  // [wave][16][kPitch], then lse_sh [wave][16]; none where tw is 1
  const int wave = wave_id(), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  // All rows' last splits first, their first ones at the end, where the short
  // rows (behind the long ones, if the caller sorts them) fill the tail.  With a
  // row's splits side by side the later (often empty) ones would fall on the
  // same XCDs for every row: workgroup b runs on XCD b % 8.
  // The waves are tw token parts of waves / tw head blocks.
  const int waves = blockDim.x >> 6, hpw = waves / a.tw, groups = (a.nhb + hpw - 1) / hpw;
  unsigned bid = blockIdx.x;
  const int hb = (int)(bid % (unsigned)groups) * hpw + wave / a.tw, tpart = wave % a.tw;
  bid /= (unsigned)groups;
  const int ri = (int)(bid % (unsigned)a.n_rows), split = a.nsplit - 1 - (int)(bid / (unsigned)a.n_rows);
  const int row = a.rows ? a.rows[ri] : ri;
  const int kv = min(a.row_pos[row], a.max_tok - 1) + 1;  // keys 0 .. kv - 1, none when <= 0
  const int* bt = a.bt + (a.row_bt ? a.row_bt[row] : row) * a.bt_stride;
  // Columns: column n is query head h0 + n, of kv head kh0 + n / group (of kh0
  // where a kv head has 16 or more).
  int kh0, h0, ncol;
  if (NH == 1 && a.group > 16) {
    const int sub = (a.group + 15) / 16;
    kh0 = hb / sub;
    h0 = kh0 * a.group + hb % sub * 16;
    ncol = min(16, (kh0 + 1) * a.group - h0);
  } else {
    kh0 = hb * NH;
    h0 = kh0 * a.group;
    ncol = min(NH, a.c.kv_heads - kh0) * a.group;
  }
  if (hb >= a.nhb) ncol = 0;
  const bool col_ok = n < ncol;
  const int my = !col_ok ? -1 : NH == 1 ? 0 : n / a.group;
  const int my_head = min(kh0 + max(my, 0), a.c.kv_heads - 1);

  bf16v8_t q[NK][QP];
#pragma unroll
  for (int s = 0; s < NK; ++s)
    load_q8<QP>(a, (int64_t)row * a.ldq + (int64_t)(h0 + n) * HD + q_dim<HD>(s, g), col_ok, 1.f, q[s]);

  float m = kLowest, l = 0.f;
  int E = 0;
  f32x4_t O[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) O[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  const int nblk = kv > 0 ? (kv + kBlk - 1) / kBlk : 0;
  const int b0 = split * a.split_blocks + tpart;
  const int b1 = ncol <= 0 ? 0 : split == a.nsplit - 1 ? nblk : min(nblk, (split + 1) * a.split_blocks);
  attend_keys<HD, NH, QP, PP, false>(a, bt, q, kv, kv - 1, kv, b0, b1, a.tw, kh0, my, my_head, col_ok, m, l, E, O);

  // Each wave's normalised output and log2 sum, then, where several waves share
  // the columns, their weighted mean.
  l = column_sum(l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float lse = l == 0.f ? -INFINITY : m - 8.f + __log2f(l);
  const int64_t part = ((int64_t)ri * a.nsplit + split) * a.n_heads + h0;
  if (a.tw == 1) {
    if (!col_ok) return;
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      float o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = ldexpf(O[i][r] * inv, E - 127);
      const int d = 16 * i + 4 * g;
      if (a.nsplit == 1) store_out4(a, (int64_t)row * a.ldo + (int64_t)(h0 + n) * HD + d, o);
      else *(float4*)(a.part + (part + n) * HD + d) = make_float4(o[0], o[1], o[2], o[3]);
    }
    if (a.nsplit > 1 && g == 0) a.lse[part + n] = lse;
    return;
  }
  float* lse_sh = o_sh + waves * 16 * kPitch;
  if (g == 0) lse_sh[wave * 16 + n] = lse;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) o_sh[(wave * 16 + n) * kPitch + 16 * i + 4 * g + r] = ldexpf(O[i][r] * inv, E - 127);
  __syncthreads();
  const int w0 = wave - tpart;
  for (int t = tpart * 64 + lane; t < ncol * (HD / 4); t += a.tw * 64) {
    const int col = t / (HD / 4), d = t % (HD / 4) * 4;
    float top = -INFINITY;
    for (int w = w0; w < w0 + a.tw; ++w) top = fmaxf(top, lse_sh[w * 16 + col]);
    float o[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
    for (int w = w0; w < w0 + a.tw; ++w) {
      const float lw = lse_sh[w * 16 + col];
      if (lw == -INFINITY) continue;
      const float f = fast_exp2(lw - top);
      sum += f;
      for (int i = 0; i < 4; ++i) o[i] += f * o_sh[(w * 16 + col) * kPitch + d + i];
    }
    const float norm = sum == 0.f ? 0.f : 1.f / sum;
    for (int i = 0; i < 4; ++i) o[i] *= norm;
    if (a.nsplit == 1) {
      store_out4(a, (int64_t)row * a.ldo + (int64_t)(h0 + col) * HD + d, o);
    } else {
      *(float4*)(a.part + (part + col) * HD + d) = make_float4(o[0], o[1], o[2], o[3]);
      if (d == 0) a.lse[part + col] = sum == 0.f ? -INFINITY : top + __log2f(sum);
    }
  }
}

// Chunks at head_dim 64 and 128.  A workgroup owns (tile, kv head, a group of its
// columns, split): column c is row c / group of the tile and query head c % group of
// the kv head's own.  Each wave has 32 columns and one of KG parts of the keys
// (KG * HD = 128), whose results are joined at the end (two heads of 64 together
// instead: 61 us for two chunks of 512 rows after 2048 x 32 heads, two parts of the
// keys 45: the work comes in smaller pieces).  KG blocks of 64 tokens (8 KB of K and
// of V) are converted to bf16 and f16 once, by all waves, into LDS in the order in
// which the products take them; while they are multiplied the next ones' codes are
// in registers, on their way from the cache.  The scales go in with the conversion:
// K's exactly, V's as 2^(byte - E + 6), so that the largest code comes to 448 * 64
// and what is lost of small slices stays below 2^-30 of the largest |V|.  The
// probabilities' sums are one more product, with a V of ones, on the rounded values
// that the outputs are made of.
//
// 512 rows after 16384, 32 / 8 heads of 128: 143 us and 10 of joining, 0.91 PFLOP/s
// (a large library product reaches 1.2).  MFMAs are busy 43% of the SIMDs' cycles
// and vector instructions 52% (per wave and block 300: the products' 68, 32 fma, 32
// exp2 at half the rate, 16 conversions, 16 max, and its share of the staging); each wave reads
// 32 KB of operands a block from LDS, half of what that delivers meanwhile.  Two
// groups of waves in alternate phases, one's products beside the other's softmax,
// change nothing (176 us both; head_dim 64 218 -> 244).
constexpr int kChunkCols = 32;  // columns of a wave at head_dim 32
// The other head dims: 16 where three parts of q of 128 dims would not leave room
// for the rest (28 / 4 heads of 128, 1024 fp32 rows after 2048: 32 columns spill
// and take 200 us, 16 101).
constexpr int chunk_cols(int hd, int qp) { return hd == 128 && qp == 3 ? 16 : kChunkCols; }

// Scores that come out of the products as log2 units against the running
// reference, s - m + 8, the sums' initial value being 8 - m and q scaled on the way
// in: no instruction per score to scale it and to subtract m.  Not for bf16 q,
// which one part holds exactly as it is, but not scaled.
constexpr bool relative_scores(int qp) { return qp > 1; }

template <bool kRel>
__device__ inline f32x4_t first_sums(float m) {
  const float x = kRel ? 8.f - m : 0.f;
  return f32x4_t{x, x, x, x};
}

// Raises a column's reference m to the block's maximum where that passes it by
// more than 2^7, and what was summed against the old one with it.  fresh: the
// column has met no score yet (above -inf); it stays so only where more keys follow,
// its last one being pos and the next block's first one `next`.
template <bool kRel, int ND, int CT>
__device__ inline void raise_reference(f32x4_t (&S)[4][CT], f32x4_t (&O)[ND][CT], f32x4_t (&l)[CT], float (&m)[CT],
                                       float qscale, bool (&fresh)[CT], const int (&pos)[CT], int next) {
  float top[CT];
  bool grow = false;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    top[ct] = -INFINITY;
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) top[ct] = fmaxf(top[ct], S[p][ct][i]);
    if constexpr (!kRel) top[ct] *= qscale;
    grow |= kRel ? fresh[ct] || top[ct] > 15.f : top[ct] > m[ct] + 7.f;
  }
  if (!__ballot(grow)) return;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const float t = column_max(top[ct]);
    float r, m1;
    if constexpr (kRel) {
      // The first reference may also be a lower one than the initial 0.
      const float up = fresh[ct] ? (t == -INFINITY ? 0.f : t - 8.f) : fmaxf(t - 8.f, 0.f);
      r = fresh[ct] ? 1.f : fast_exp2(-up);
      m1 = m[ct] + up;
      fresh[ct] = fresh[ct] && t == -INFINITY && pos[ct] >= next;
#pragma unroll
      for (int p = 0; p < 4; ++p) S[p][ct] -= up;
    } else {
      m1 = fmaxf(m[ct], t);
      r = fast_exp2(m[ct] - m1);
    }
    l[ct] *= r;
#pragma unroll
    for (int i = 0; i < ND; ++i) O[i][ct] *= r;
    m[ct] = m1;
  }
}

template <int HD>
struct ChunkStage {
  static constexpr int KG = 128 / HD;
  u32x4_t k[KG][4][HD / 32][64];  // [block][product][k step][lane] 8 bf16
  u32x4_t v[KG][HD / 16][2][64];  // [block][dims][half][lane] 8 f16
  int E[KG];                      // the largest V byte so far of the part
  uint64_t bad[KG];               // tokens whose V slice is NaN
};

// LDS of a workgroup of the chunk kernel: two stages and the waves' V factors,
// and at the end, in the same place, the parts' results.
template <int HD>
constexpr size_t chunk_lds(int waves) {
  const size_t stages = 2 * sizeof(ChunkStage<HD>) + waves * 64 * sizeof(_Float16);
  const size_t join = (size_t)waves * (HD == 128 ? 16 : 32) * (HD + 5) * sizeof(float);  // 128: of few columns
  return stages > join ? stages : join;
}

// A tile of few columns (the last rows of a prompt, a short turn after a long one):
// its W waves are parts of the keys, 16 columns each, straight from the cache like the
// single rows.  In the other way the waves past the columns would only convert for the
// rest.  us, that way / this one:
//   16 heads of 128, 8 rows after 16384     40 / 25    32 heads of 64  32 / 22
//   32 / 8 heads of 128, 4 rows after 4096  17 / 15, 8 after 1000  14.4 / 13.1, and of
//     more than 32 columns, 14 rows after 16384  29 / 36: each wave converts for 16
//     columns only
constexpr int kFewCols = 32;

template <int HD, int W, int QP, int PP, typename Finish>
__device__ __forceinline__ void few_columns(const AttnArgs& a, const int* bt, float* o_sh, int kh, int split, int cols,
                                            int row0, int pos0, Finish finish) {
  constexpr int NK = HD / 32, ND = HD / 16, kPitch = HD + 4;
  const int wave = wave_id(), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  int cw = 1;  // waves that the columns take
  while (16 * cw < cols) cw *= 2;
  const int parts = W / cw, part = wave / cw, c0 = wave % cw * 16, c = c0 + n;
  const bool col_ok = c < cols;
  const int t = c / a.group, pos = col_ok ? min(pos0 + t, a.max_tok - 1) : -1;
  bf16v8_t q[NK][QP];
#pragma unroll
  for (int s = 0; s < NK; ++s)
    load_q8<QP>(a, (int64_t)(row0 + t) * a.ldq + (int64_t)(kh * a.group + c % a.group) * HD + q_dim<HD>(s, g), col_ok, 1.f, q[s]);
  const int kv = c0 < cols ? min(pos0 + (min(c0 + 16, cols) - 1) / a.group, a.max_tok - 1) + 1 : 0;
  const int nblk = kv > 0 ? (kv + kBlk - 1) / kBlk : 0;
  const int b0 = split * a.split_blocks + part;
  const int b1 = split == a.nsplit - 1 ? nblk : min(nblk, (split + 1) * a.split_blocks);
  float m = kLowest, l = 0.f;
  int E = 0;
  f32x4_t O[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) O[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  attend_keys<HD, 1, QP, PP, true>(a, bt, q, kv, pos, min(pos0 + c0 / a.group, a.max_tok - 1) + 1, b0, b1, parts, kh, 0,
                                   kh, col_ok, m, l, E, O);

  l = column_sum(l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float* lse_sh = o_sh + W * 16 * kPitch;
  if (g == 0) lse_sh[wave * 16 + n] = l == 0.f ? -INFINITY : m - 8.f + __log2f(l);
#pragma unroll
  for (int i = 0; i < ND; ++i)
    *(float4*)(o_sh + (wave * 16 + n) * kPitch + 16 * i + 4 * g) =
        make_float4(ldexpf(O[i][0] * inv, E - 127), ldexpf(O[i][1] * inv, E - 127), ldexpf(O[i][2] * inv, E - 127),
                    ldexpf(O[i][3] * inv, E - 127));
  __syncthreads();
  for (int i = threadIdx.x; i < cols * (HD / 4); i += W * 64) {
    const int col = i / (HD / 4), d = i % (HD / 4) * 4;
    float top = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int x = 0; x < parts; ++x) top = fmaxf(top, lse_sh[x * cw * 16 + col]);
    for (int x = 0; x < parts; ++x) {
      const float lw = lse_sh[x * cw * 16 + col];
      if (lw == -INFINITY) continue;
      const float f = fast_exp2(lw - top);
      const float4 y = *(const float4*)(o_sh + (x * cw * 16 + col) * kPitch + d);
      sum += f;
      o[0] += f * y.x; o[1] += f * y.y; o[2] += f * y.z; o[3] += f * y.w;
    }
    const float norm = sum == 0.f ? 0.f : 1.f / sum;
    for (int e = 0; e < 4; ++e) o[e] *= norm;
    finish(col, d, o, sum == 0.f ? -INFINITY : top + __log2f(sum));
  }
}

template <int HD, int SW, int QP, int PP>
__global__ __launch_bounds__(512 / SW) void kv8_chunk_kernel(const AttnArgs a) {
  constexpr int NK = HD / 32, ND = HD / 16, KG = 128 / HD, W = 8 / SW, WH = W / KG, COLS = chunk_cols(HD, QP), CT = COLS / 16;
  constexpr bool kRel = relative_scores(QP);
  extern __shared__ __align__(16) char lds[];
  ChunkStage<HD>* stage = (ChunkStage<HD>*)lds;
  _Float16(*factor)[64] = (_Float16(*)[64])(lds + 2 * sizeof(ChunkStage<HD>));  // a wave's own, of the block it stages
  const int wave = wave_id(), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  unsigned unit = blockIdx.x;
  const int cg = (int)(unit % (unsigned)a.ncg);
  unit /= (unsigned)a.ncg;
  const int kh = (int)(unit % (unsigned)a.c.kv_heads);
  unit /= (unsigned)a.c.kv_heads;
  const int split = (int)(unit % (unsigned)a.nsplit);
  const int64_t tile = unit / (unsigned)a.nsplit;
  // Tiles are handed over as cbis_paged_prefill_attention's: row, rows, table row,
  // position (past the table all are alike: every key it covers).
  const int row0 = a.tiles[4 * tile], nv = min(a.tiles[4 * tile + 1], CBIS_PREFILL_TILE_ROWS),
            btr = a.tiles[4 * tile + 2], pos0 = min(a.tiles[4 * tile + 3], a.max_tok);
  const int cols = nv * a.group, wg0 = cg * WH * COLS;
  if (wg0 >= cols) return;
  const int* bt = a.bt + (int64_t)btr * a.bt_stride;
  // A column's result: normalised outputs and the log2 of its sum.
  auto finish = [&](int c, int d, const float* o, float lse) {
    const int t = c / a.group, head = kh * a.group + c % a.group;
    if (a.nsplit == 1) {
      store_out4(a, (int64_t)(row0 + t) * a.ldo + (int64_t)head * HD + d, o);
    } else {
      const int64_t at = ((tile * CBIS_PREFILL_TILE_ROWS + t) * a.nsplit + split) * a.n_heads + head;
      *(float4*)(a.part + at * HD + d) = make_float4(o[0], o[1], o[2], o[3]);
      if (d == 0) a.lse[at] = lse;
    }
  };
  if (cols <= (W < 4 || COLS < 32 ? 16 : kFewCols)) {
    few_columns<HD, W, QP, PP>(a, bt, (float*)lds, kh, split, cols, row0, pos0, finish);
    return;
  }
  const int H = a.c.kv_heads, j = wave / WH;  // j: the wave's part of the keys
  const int c0 = wg0 + wave % WH * COLS;
  const bool busy = c0 < cols;  // the others stage only
  const int first_pos = min(pos0 + c0 / a.group, a.max_tok - 1);
  const int last_pos = min(pos0 + (min(c0 + COLS, cols) - 1) / a.group, a.max_tok - 1);
  int pos[CT];
  bf16v8_t q[CT][NK][QP];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = c0 + 16 * ct + n, t = c / a.group, head = kh * a.group + c % a.group;
    const bool ok = busy && c < cols;
    pos[ct] = ok ? min(pos0 + t, a.max_tok - 1) : -1;
#pragma unroll
    for (int s = 0; s < NK; ++s)
      load_q8<QP>(a, (int64_t)(row0 + t) * a.ldq + (int64_t)head * HD + q_dim<HD>(s, g), ok, kRel ? a.qscale : 1.f, q[ct][s]);
  }
  float m[CT];
  bool fresh[CT];
  int E = 0;
  f32x4_t O[ND][CT], l[CT];  // l: every lane of a column holds its sum four times over
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = kRel ? 0.f : kLowest;
    fresh[ct] = true;
    l[ct] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < ND; ++i) O[i][ct] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  f16v8_t ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = (_Float16)1.f;
  // The workgroup's keys.
  const int kv = min(pos0 + (min(wg0 + WH * COLS, cols) - 1) / a.group, a.max_tok - 1) + 1;
  const int nblk = kv > 0 ? (kv + kBlk - 1) / kBlk : 0;
  const int b0 = split * a.split_blocks;
  const int b1 = split == a.nsplit - 1 ? nblk : min(nblk, b0 + a.split_blocks);
  const int tlast = (kv - 1) >> 4;
  const int rounds = (b1 - b0 + KG - 1) / KG;
  const int64_t codes = (int64_t)H * HD * kTile;
  const int64_t head_codes = (int64_t)kh * HD * kTile, head_bytes = codes + kh * kTile;

  // Staging: item f = wave * SW + i of 8 is 64 lanes' 16 bytes of K and of V.
  const int js = HD == 128 ? 0 : wave * SW >> 2;  // the part whose blocks the wave stages
  auto block_of = [&](int r, int part) { return b0 + r * KG + part; };
  auto k_tile = [&](int r) { return min(4 * block_of(r, js) + (n >> 2), tlast); };
  auto v_tile = [&](int r) { return min(4 * block_of(r, js) + g, tlast); };
  int kpage, vpage;  // of the lane's tiles of the block to load, read a round ahead
  u32x4_t kraw[SW], vraw[SW];
  // Scale bytes come as the dwords that hold them: taken out of a byte load they
  // would be awaited where the load is issued.
  uint32_t kbyte[SW], vbyte = 0;
  int Es = 0;  // the largest V byte so far of that part
  auto load_block = [&](int b) {
    const int64_t ko = tile_offset(a.c, kpage, k_tile(b)), vo = tile_offset(a.c, vpage, v_tile(b));
    kpage = bt[k_tile(b + 1) >> a.c.tshift];
    vpage = bt[v_tile(b + 1) >> a.c.tshift];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < SW; ++i) {
      const int f = wave * SW + i;
      const uint8_t* kp = a.c.k + ko + head_codes + (n & 3) * HD;
      const uint32_t* kb = (const uint32_t*)(a.c.k + ko + head_bytes);
      const int p = HD == 64 ? f & 3 : f >> 1, h = HD == 64 ? 0 : f & 1, dt = HD == 64 ? f & 3 : f;
      kraw[i] = *(const u32x4_t*)(kp + 4 * p * HD + 16 * g + 64 * h);
      kbyte[i] = kb[p];
      vraw[i] = *(const u32x4_t*)(a.c.v + vo + head_codes + (dt * 16 + n) * kTile);
    }
    vbyte = *(const uint32_t*)(a.c.v + vo + head_bytes + (n & 12));
    __builtin_amdgcn_sched_barrier(0);
  };
  auto store_block = [&](int r, ChunkStage<HD>& st) {
    const int b = block_of(r, js);
    const int valid = min(max(kv - (b * kBlk + g * kTile), 0), kTile);  // tokens of tile g that may be seen
    const bool tail = (b + 1) * kBlk > kv;
    // The V factors: a lane makes token 16 g + n's, and takes tile g's 16.
    int byte = n < valid ? (int)byte_of(vbyte, n & 3) : 0;
    const uint64_t bad = __ballot(byte == kBadByte);
    if (byte == kBadByte) byte = 0;
    if (__ballot(byte > Es)) {
      int top = max(byte, Es);
#pragma unroll
      for (int x = 1; x < 64; x *= 2) top = max(top, __shfl_xor(top, x, 64));
      Es = __builtin_amdgcn_readfirstlane(top);
    }
    factor[wave][lane] = (_Float16)ldexpf(1.f, byte - Es + 6);
    if (lane == 0) {  // the waves of a part write the same
      st.E[js] = Es;
      st.bad[js] = bad;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const f16v8_t f0 = *(const f16v8_t*)&factor[wave][16 * g], f1 = *(const f16v8_t*)&factor[wave][16 * g + 8];
#pragma unroll
    for (int i = 0; i < SW; ++i) {
      const int f = wave * SW + i;
      const int p = HD == 64 ? f & 3 : f >> 1, h = HD == 64 ? 0 : f & 1, dt = HD == 64 ? f & 3 : f;
      const float scale = pow2_of_byte(byte_of(kbyte[i], n & 3));  // 255: NaN scores
      st.k[js][p][2 * h][lane] = __builtin_bit_cast(u32x4_t, codes_bf16(kraw[i][0], kraw[i][1], scale));
      st.k[js][p][2 * h + 1][lane] = __builtin_bit_cast(u32x4_t, codes_bf16(kraw[i][2], kraw[i][3], scale));
      u32x4_t w = vraw[i];
      if (tail) {  // a slot past the last key may hold anything
#pragma unroll
        for (int d = 0; d < 4; ++d) w[d] &= token_mask(valid, d);
      }
      st.v[js][dt][0][lane] = __builtin_bit_cast(u32x4_t, codes_f16(w[0], w[1]) * f0);
      st.v[js][dt][1][lane] = __builtin_bit_cast(u32x4_t, codes_f16(w[2], w[3]) * f1);
    }
  };

  if (rounds > 0) {
    kpage = bt[k_tile(0) >> a.c.tshift];
    vpage = bt[v_tile(0) >> a.c.tshift];
    load_block(0);
    store_block(0, stage[0]);
    load_block(1);
    lds_barrier();
  }
  for (int r = 0; r < rounds; ++r) {
    const ChunkStage<HD>& st = stage[r & 1];
    const int b = block_of(r, j);
    if (busy && b < b1 && b * kBlk <= last_pos) {
      // Operands come from LDS four at a time, the next four before these are
      // used (left to itself the compiler reads each just ahead of its product).
      f32x4_t S[4][CT];
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) S[p][ct] = first_sums<kRel>(m[ct]);
      // Operand y is product op_p(y), k step op_s(y): products alternate, so that no
      // two instructions in a row wait for the same sums.
      auto op_p = [](int y) { return y / (2 * NK) * 2 + (y & 1); };
      auto op_s = [](int y) { return y % (2 * NK) / 2; };
      bf16v8_t kf[2][4];
#pragma unroll
      for (int x = 0; x < 4; ++x) kf[0][x] = __builtin_bit_cast(bf16v8_t, st.k[j][op_p(x)][op_s(x)][lane]);
#pragma unroll
      for (int y = 0; y < NK; ++y) {
        if (y + 1 < NK) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            kf[(y + 1) & 1][x] = __builtin_bit_cast(bf16v8_t, st.k[j][op_p(4 * y + 4 + x)][op_s(4 * y + 4 + x)][lane]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < QP; ++k)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int p = op_p(4 * y + x), s = op_s(4 * y + x);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
              S[p][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[y & 1][x], q[ct][s][k], S[p][ct], 0, 0, 0);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
      constexpr int GV = 4, NG = ND / GV;  // V operands of a group, groups of a half
      f16v8_t vf[2][GV];
      auto load_vf = [&](int y) {
#pragma unroll
        for (int x = 0; x < GV; ++x)
          vf[y & 1][x] = __builtin_bit_cast(f16v8_t, st.v[j][y % NG * GV + x][y / NG][lane]);
      };
      load_vf(0);
      const int t0 = b * kBlk + g * kTile;  // first token of the lane's tile
      if ((b + 1) * kBlk > first_pos + 1) {
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
              if (t0 + 4 * p + i > pos[ct]) S[p][ct][i] = -INFINITY;
      }
      const uint64_t bad = st.bad[j];
      if (bad) {  // a column that sees a V slice of NaN becomes NaN
        const unsigned mine = (unsigned)(bad >> (16 * g));
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
              if ((mine & (1u << (4 * p + i))) && S[p][ct][i] != -INFINITY) S[p][ct][i] = NAN;
      }
      const int E1 = __builtin_amdgcn_readfirstlane(st.E[j]);
      if (E1 != E) {
        const float r = ldexpf(1.f, E - E1);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int i = 0; i < ND; ++i) O[i][ct] *= r;
        E = E1;
      }
      raise_reference<kRel, ND, CT>(S, O, l, m, a.qscale, fresh, pos, (b + 1) * kBlk);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        f16v8_t P[CT][PP];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float x = fast_exp2(kRel ? S[2 * half + h][ct][i] : S[2 * half + h][ct][i] * a.qscale - (m[ct] - 8.f));
#pragma unroll
              for (int k = 0; k < PP; ++k) {
                const _Float16 y = (_Float16)x;
                P[ct][k][4 * h + i] = y;
                x -= (float)y;
              }
            }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int k = 0; k < PP; ++k) l[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, P[ct][k], l[ct], 0, 0, 0);
#pragma unroll
        for (int y = half * NG; y < half * NG + NG; ++y) {
          if (y + 1 < 2 * NG) load_vf(y + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int k = 0; k < PP; ++k)
#pragma unroll
            for (int x = 0; x < GV; ++x)
#pragma unroll
              for (int ct = 0; ct < CT; ++ct)
                O[y % NG * GV + x][ct] =
                    __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[y & 1][x], P[ct][k], O[y % NG * GV + x][ct], 0, 0, 0);
        }
      }
    }
    if (r + 1 < rounds) {
      store_block(r + 1, stage[(r + 1) & 1]);
      load_block(r + 2);  // behind the last block: the last tile again
      lds_barrier();
    }
  }
  constexpr int kPitch = HD + 4, WC = WH * COLS;
  float* o_sh = (float*)lds;                 // [part][column][kPitch]
  float* lse_sh = o_sh + KG * WC * kPitch;   // [part][column]
  if constexpr (KG > 1) __syncthreads();     // the last round's operands have been read
  if (busy) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int c = c0 + 16 * ct + n;
      const float sum = l[ct][0], inv = sum == 0.f ? 0.f : 1.f / sum;
      const float lse = sum == 0.f ? -INFINITY : m[ct] - 8.f + __log2f(sum);
      if (KG > 1 && g == 0) lse_sh[j * WC + c - wg0] = lse;
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        float o[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) o[x] = ldexpf(O[i][ct][x] * inv, E - 133);
        const int d = 16 * i + 4 * g;
        if constexpr (KG > 1) *(float4*)(o_sh + (j * WC + c - wg0) * kPitch + d) = make_float4(o[0], o[1], o[2], o[3]);
        else if (c < cols) finish(c, d, o, lse);
      }
    }
  }
  if constexpr (KG > 1) {
    __syncthreads();
    for (int t = threadIdx.x; t < min(cols - wg0, WC) * (HD / 4); t += W * 64) {
      const int c = t / (HD / 4), d = t % (HD / 4) * 4;
      float top = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < KG; ++x) top = fmaxf(top, lse_sh[x * WC + c]);
#pragma unroll
      for (int x = 0; x < KG; ++x) {
        const float lw = lse_sh[x * WC + c];
        if (lw == -INFINITY) continue;
        const float f = fast_exp2(lw - top);
        const float4 y = *(const float4*)(o_sh + (x * WC + c) * kPitch + d);
        sum += f;
        o[0] += f * y.x; o[1] += f * y.y; o[2] += f * y.z; o[3] += f * y.w;
      }
      const float norm = sum == 0.f ? 0.f : 1.f / sum;
      for (int i = 0; i < 4; ++i) o[i] *= norm;
      finish(wg0 + c, d, o, sum == 0.f ? -INFINITY : top + __log2f(sum));
    }
  }
}

// Chunks at head_dim 32, where K and V are cheap to convert and the softmax is
// everything: a wave has 32 columns of a kv head and every tw-th block of 64
// tokens, straight from the cache through registers like the single rows'
// kernel, so that waves run apart and fill each other's gaps.
//
// Two chunks of 512 rows after 0 and 512, 64 heads: 21.9 us, of 2048 waves with 1 to
// 16 blocks each; 512 rows after 16384: 183.  Vector instructions are issued in
// 63% of the SIMDs' cycles (some 310 for a block's 32 columns, 32 of them exp2 at
// half the rate, by the counters), products in 20%.
template <int QP, int PP>
__global__ __launch_bounds__(kDecodeWaves * 64) void kv8_chunk32_kernel(const AttnArgs a) {
  constexpr int HD = 32, ND = 2, CT = kChunkCols / 16, kPitch = HD + 4;
  constexpr bool kRel = relative_scores(QP);
  // Per wave 64 V factors of the block at hand; at the end the parts' results.
  extern __shared__ __align__(16) char lds[];
  const int wave = wave_id(), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int waves = blockDim.x >> 6, upw = waves / a.tw, tpart = wave % a.tw;  // upw: units of a workgroup
  unsigned unit = blockIdx.x * (unsigned)upw + wave / a.tw;
  const int cg = (int)(unit % (unsigned)a.ncg);
  unit /= (unsigned)a.ncg;
  const int kh = (int)(unit % (unsigned)a.c.kv_heads);
  unit /= (unsigned)a.c.kv_heads;
  const int split = (int)(unit % (unsigned)a.nsplit);
  const int tile = (int)(unit / (unsigned)a.nsplit);
  const bool in = tile < a.n_tiles;
  const int4 td = in ? *(const int4*)(a.tiles + 4 * (int64_t)tile) : make_int4(0, 0, 0, 0);
  const int row0 = td.x, nv = min(td.y, CBIS_PREFILL_TILE_ROWS), pos0 = min(td.w, a.max_tok);
  const int c0 = cg * kChunkCols, cols = nv * a.group;
  const bool busy = in && c0 < cols;
  const int* bt = a.bt + (int64_t)td.z * a.bt_stride;
  const int first_pos = min(pos0 + c0 / a.group, a.max_tok - 1);
  const int last_pos = min(pos0 + (min(c0 + kChunkCols, cols) - 1) / a.group, a.max_tok - 1);
  int pos[CT];
  bf16v8_t q[CT][QP];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = c0 + 16 * ct + n, t = c / a.group, head = kh * a.group + c % a.group;
    const bool ok = busy && c < cols;
    pos[ct] = ok ? min(pos0 + t, a.max_tok - 1) : -1;
    load_q8<QP>(a, (int64_t)(row0 + t) * a.ldq + (int64_t)head * HD + q_dim<HD>(0, g), ok, kRel ? a.qscale : 1.f, q[ct]);
  }
  float m[CT];
  bool fresh[CT];
  int E = 0;
  f32x4_t O[ND][CT], l[CT];  // l: every lane of a column holds its sum four times over
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = kRel ? 0.f : kLowest;
    fresh[ct] = true;
    l[ct] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < ND; ++i) O[i][ct] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  f16v8_t ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = (_Float16)1.f;

  const int kv = last_pos + 1;
  const int nblk = busy && kv > 0 ? (kv + kBlk - 1) / kBlk : 0;
  const int b0 = split * a.split_blocks + tpart;
  const int b1 = split == a.nsplit - 1 ? nblk : min(nblk, (split + 1) * a.split_blocks);
  const int tlast = (kv - 1) >> 4;
  const int64_t codes = (int64_t)a.c.kv_heads * HD * kTile;
  const int64_t k_off = (int64_t)kh * HD * kTile + (n & 3) * HD + 8 * g, v_off = (int64_t)kh * HD * kTile + n * kTile;
  const int64_t byte_off = codes + kh * kTile;
  _Float16* factor = (_Float16*)lds + wave * 64;

  if (b0 < b1) {
    auto k_tile = [&](int b) { return min(4 * b + (n >> 2), tlast); };
    auto v_tile = [&](int b) { return min(4 * b + g, tlast); };
    KRaw<HD> kr[4];
    u32x4_t vr[ND], kb;
    uint32_t vbyte;
    auto load_k_block = [&](int64_t at) {
#pragma unroll
      for (int p = 0; p < 4; ++p) kr[p] = load_k<HD>(a.c.k + at + k_off + 4 * p * HD);
      kb = *(const u32x4_t*)(a.c.k + at + byte_off);
    };
    auto load_v_block = [&](int64_t at) {
      vbyte = *(const uint32_t*)(a.c.v + at + byte_off + (n & 12));
#pragma unroll
      for (int i = 0; i < ND; ++i) vr[i] = *(const u32x4_t*)(a.c.v + at + v_off + i * kTile * kTile);
    };
    const int kpage0 = bt[k_tile(b0) >> a.c.tshift], vpage0 = bt[v_tile(b0) >> a.c.tshift];
    int kpage = bt[k_tile(b0 + a.tw) >> a.c.tshift], vpage = bt[v_tile(b0 + a.tw) >> a.c.tshift];
    load_k_block(tile_offset(a.c, kpage0, k_tile(b0)));
    load_v_block(tile_offset(a.c, vpage0, v_tile(b0)));
    for (int b = b0; b < b1; b += a.tw) {
      f32x4_t S[4][CT];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float ks = pow2_of_byte(byte_of(kb[p], n & 3));  // 255: NaN scores
        const bf16v8_t kf = codes_bf16(kr[p].w[0], kr[p].w[1], ks);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          S[p][ct] = first_sums<kRel>(m[ct]);
#pragma unroll
          for (int k = 0; k < QP; ++k)
            S[p][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[ct][k], S[p][ct], 0, 0, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      load_k_block(tile_offset(a.c, kpage, k_tile(b + a.tw)));
      __builtin_amdgcn_sched_barrier(0);
      const int t0 = b * kBlk + g * kTile;  // first token of the lane's tile
      if ((b + 1) * kBlk > first_pos + 1) {
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
              if (t0 + 4 * p + i > pos[ct]) S[p][ct][i] = -INFINITY;
      }
      // V's factors: a lane makes token 16 g + n's, and takes tile g's 16.
      const int valid = min(max(kv - t0, 0), kTile);  // tokens of tile g that may be seen
      int byte = n < valid ? (int)byte_of(vbyte, n & 3) : 0;
      const uint64_t bad = __ballot(byte == kBadByte);
      if (bad) {  // a column that sees a V slice of NaN becomes NaN
        if (byte == kBadByte) byte = 0;
        const unsigned mine = (unsigned)(bad >> (16 * g));
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
              if ((mine & (1u << (4 * p + i))) && S[p][ct][i] != -INFINITY) S[p][ct][i] = NAN;
      }
      if (__ballot(byte > E)) {
        int E1 = max(byte, E);
#pragma unroll
        for (int x = 1; x < 64; x *= 2) E1 = max(E1, __shfl_xor(E1, x, 64));
        E1 = __builtin_amdgcn_readfirstlane(E1);
        const float r = ldexpf(1.f, E - E1);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int i = 0; i < ND; ++i) O[i][ct] *= r;
        E = E1;
      }
      factor[lane] = (_Float16)ldexpf(1.f, byte - E + 6);
      raise_reference<kRel, ND, CT>(S, O, l, m, a.qscale, fresh, pos, (b + 1) * kBlk);
      if ((b + 1) * kBlk > kv) {  // a slot past the last key may hold anything
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const uint32_t mask = token_mask(valid, d);
#pragma unroll
          for (int i = 0; i < ND; ++i) vr[i][d] &= mask;
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const f16v8_t f = *(const f16v8_t*)(factor + 16 * g + 8 * half);
        f16v8_t P[CT][PP];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float y0 = S[2 * half + i / 4][ct][i & 3];
            float x = fast_exp2(kRel ? y0 : y0 * a.qscale - (m[ct] - 8.f));
#pragma unroll
            for (int k = 0; k < PP; ++k) {
              const _Float16 y = (_Float16)x;
              P[ct][k][i] = y;
              x -= (float)y;
            }
          }
#pragma unroll
        for (int k = 0; k < PP; ++k)
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            l[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, P[ct][k], l[ct], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < ND; ++i)
              O[i][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16(vr[i][2 * half], vr[i][2 * half + 1]) * f,
                                                                P[ct][k], O[i][ct], 0, 0, 0);
          }
      }
      __builtin_amdgcn_sched_barrier(0);
      const int64_t vo = tile_offset(a.c, vpage, v_tile(b + a.tw));
      kpage = bt[k_tile(b + 2 * a.tw) >> a.c.tshift];
      vpage = bt[v_tile(b + 2 * a.tw) >> a.c.tshift];
      __builtin_amdgcn_sched_barrier(0);
      load_v_block(vo);  // behind the last block: the last tile again
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  auto finish = [&](int c, int d, const float* o, float lse) {
    const int t = c / a.group, head = kh * a.group + c % a.group;
    if (a.nsplit == 1) {
      store_out4(a, (int64_t)(row0 + t) * a.ldo + (int64_t)head * HD + d, o);
    } else {
      const int64_t at = (((int64_t)tile * CBIS_PREFILL_TILE_ROWS + t) * a.nsplit + split) * a.n_heads + head;
      *(float4*)(a.part + at * HD + d) = make_float4(o[0], o[1], o[2], o[3]);
      if (d == 0) a.lse[at] = lse;
    }
  };
  float* o_sh = (float*)lds;  // [wave][column][kPitch]
  float* lse_sh = o_sh + waves * kChunkCols * kPitch;
  if (a.tw > 1) __syncthreads();
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = c0 + 16 * ct + n;
    const float sum = l[ct][0], inv = sum == 0.f ? 0.f : 1.f / sum;
    const float lse = sum == 0.f ? -INFINITY : m[ct] - 8.f + __log2f(sum);
    if (a.tw > 1 && g == 0) lse_sh[wave * kChunkCols + 16 * ct + n] = lse;
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      float o[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) o[x] = ldexpf(O[i][ct][x] * inv, E - 133);
      const int d = 16 * i + 4 * g;
      if (a.tw > 1) *(float4*)(o_sh + (wave * kChunkCols + 16 * ct + n) * kPitch + d) = make_float4(o[0], o[1], o[2], o[3]);
      else if (busy && c < cols) finish(c, d, o, lse);
    }
  }
  if (a.tw == 1) return;
  __syncthreads();
  if (!busy) return;
  for (int t = tpart * 64 + lane; t < min(cols - c0, kChunkCols) * (HD / 4); t += a.tw * 64) {
    const int c = t / (HD / 4), d = t % (HD / 4) * 4, w0 = wave - tpart;
    float top = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int x = w0; x < w0 + a.tw; ++x) top = fmaxf(top, lse_sh[x * kChunkCols + c]);
    for (int x = w0; x < w0 + a.tw; ++x) {
      const float lw = lse_sh[x * kChunkCols + c];
      if (lw == -INFINITY) continue;
      const float f = fast_exp2(lw - top);
      const float4 y = *(const float4*)(o_sh + (x * kChunkCols + c) * kPitch + d);
      sum += f;
      o[0] += f * y.x; o[1] += f * y.y; o[2] += f * y.z; o[3] += f * y.w;
    }
    const float norm = sum == 0.f ? 0.f : 1.f / sum;
    for (int i = 0; i < 4; ++i) o[i] *= norm;
    finish(c0 + c, d, o, sum == 0.f ? -INFINITY : top + __log2f(sum));
  }
}

// The splits of a row's head joined: the mean of their outputs weighted by
// their sums.  HD / 4 lanes hold 4 dims each; `share` such groups of a wave (a
// power of two) take a (slot, head)'s splits in turn, a slot being a decode row
// or a tile's row.  Bound by latency, so that the loads of four splits go out
// together (64 rows after 16384 x 29 splits of 32 heads of 128, with the attention:
// 47.5 -> 42 us); 512 rows x 4 splits of 32 heads, 34 MB, take 10 us.
constexpr int kMergeAhead = 4;  // splits whose loads a lane has on their way

template <int HD>
__global__ __launch_bounds__(256) void kv8_merge_kernel(const AttnArgs a, int64_t slots, int share) {
  constexpr int L = HD / 4;
  const int lane = threadIdx.x & 63, d = lane % L * 4, w = L * share;
  const int64_t sh = ((int64_t)blockIdx.x * 256 + threadIdx.x) / w;
  const int head = (int)(sh % a.n_heads);
  const int64_t slot = sh / a.n_heads;
  bool ok = slot < slots;
  int64_t row = 0;
  if (ok && a.tiles) {
    const int64_t tile = slot / CBIS_PREFILL_TILE_ROWS;
    const int t = (int)(slot % CBIS_PREFILL_TILE_ROWS);
    ok = t < a.tiles[4 * tile + 1];
    row = (int64_t)a.tiles[4 * tile] + t;
  } else if (ok) {
    row = a.rows ? a.rows[slot] : slot;
  }
  const int64_t first = slot * a.nsplit * a.n_heads + head;
  // Each group's own running maximum, its sum and its weighted outputs.
  float top = -INFINITY, sum = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = lane % w / L; ok && s0 < a.nsplit; s0 += kMergeAhead * share) {
    float ls[kMergeAhead];
    f32x4_t x[kMergeAhead];
#pragma unroll
    for (int u = 0; u < kMergeAhead; ++u) {
      const int s = s0 + u * share;
      const int64_t at = first + (int64_t)min(s, a.nsplit - 1) * a.n_heads;
      ls[u] = s < a.nsplit ? a.lse[at] : -INFINITY;
      x[u] = *(const f32x4_t*)(a.part + at * HD + d);
    }
#pragma unroll
    for (int u = 0; u < kMergeAhead; ++u) {
      if (ls[u] == -INFINITY) continue;  // an empty split; its outputs may not be there
      const float t1 = fmaxf(top, ls[u]);
      const float f0 = fast_exp2(top - t1), f1 = fast_exp2(ls[u] - t1);
      sum = sum * f0 + f1;
      o = o * f0 + x[u] * f1;
      top = t1;
    }
  }
  float all = top;
  for (int x = L; x < w; x *= 2) all = fmaxf(all, __shfl_xor(all, x, 64));
  const float f = sum == 0.f ? 0.f : fast_exp2(top - all);
  sum *= f;
  o *= f;
  for (int x = L; x < w; x *= 2) {
    sum += __shfl_xor(sum, x, 64);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x, 64);
  }
  if (!ok || lane % w >= L) return;
  const float norm = sum == 0.f ? 0.f : 1.f / sum;
  const float out[4] = {o[0] * norm, o[1] * norm, o[2] * norm, o[3] * norm};
  store_out4(a, row * a.ldo + (int64_t)head * HD + d, out);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
bool geometry_ok(int kv_heads, int head_dim, int page_size) {
  return kv_heads > 0 && (head_dim == 32 || head_dim == 64 || head_dim == 128) && page_size >= kTile &&
         (page_size & (page_size - 1)) == 0;
}

int make_pages(const cbis_kv8_cache* c, Pages* p, const char* who) {
  CBIS_REQUIRE(c, CBIS_ERR_INVALID, "%s: null cache", who);
  CBIS_REQUIRE(c->n_kv_heads > 0 && c->num_pages > 0, CBIS_ERR_INVALID, "%s: n_kv_heads %d, num_pages %d", who,
               c->n_kv_heads, c->num_pages);
  CBIS_REQUIRE(geometry_ok(c->n_kv_heads, c->head_dim, c->page_size), CBIS_ERR_UNSUPPORTED,
               "%s: head_dim %d (32, 64 or 128), page_size %d (a power of two, at least 16)", who, c->head_dim,
               c->page_size);
  CBIS_REQUIRE(c->k_pool && c->v_pool && (((uintptr_t)c->k_pool | (uintptr_t)c->v_pool) & 15u) == 0, CBIS_ERR_INVALID,
               "%s: the pools must be 16-byte aligned device pointers", who);
  p->k = (uint8_t*)c->k_pool;
  p->v = (uint8_t*)c->v_pool;
  p->num_pages = c->num_pages;
  p->page_size = c->page_size;
  p->tshift = 0;
  while ((kTile << p->tshift) < c->page_size) ++p->tshift;
  p->kv_heads = c->n_kv_heads;
  p->head_dim = c->head_dim;
  p->tile_bytes = (int64_t)kTile * c->n_kv_heads * (c->head_dim + 1);
  return CBIS_OK;
}

template <typename T, int HD>
void rows_launch(bool gather, int rows, const RowsArgs& a, unsigned grid, hipStream_t s) {
  const int threads = kRowThreads / rows;
  if constexpr (HD <= 16 * kLaneCols<T>) {
    if (rows == 4 && gather) return kv8_gather_kernel<T, HD, 4><<<grid, threads, 0, s>>>(a);
    if (rows == 4) return kv8_scatter_kernel<T, HD, 4><<<grid, threads, 0, s>>>(a);
  }
  if (rows == 2 && gather) kv8_gather_kernel<T, HD, 2><<<grid, threads, 0, s>>>(a);
  else if (rows == 2) kv8_scatter_kernel<T, HD, 2><<<grid, threads, 0, s>>>(a);
  else if (gather) kv8_gather_kernel<T, HD, 1><<<grid, threads, 0, s>>>(a);
  else kv8_scatter_kernel<T, HD, 1><<<grid, threads, 0, s>>>(a);
}

template <typename T>
void rows_launch(bool gather, const RowsArgs& a, unsigned grid, hipStream_t s) {
  const int width = a.c.kv_heads * a.c.head_dim, rows = width <= 16 * kLaneCols<T> ? 4 : width <= 32 * kLaneCols<T> ? 2 : 1;
  if (a.c.head_dim == 32) rows_launch<T, 32>(gather, rows, a, grid, s);
  else if (a.c.head_dim == 64) rows_launch<T, 64>(gather, rows, a, grid, s);
  else rows_launch<T, 128>(gather, rows, a, grid, s);
}

int kv8_rows(bool gather, const cbis_kv8_cache* c, int n_rows, int dtype, const void* K, int64_t ldk, const void* V,
             int64_t ldv, const int* page, const int* offset, hipStream_t s, const char* who) {
  RowsArgs a = {};
  const int rc = make_pages(c, &a.c, who);
  if (rc) return rc;
  CBIS_REQUIRE(n_rows >= 0, CBIS_ERR_INVALID, "%s: n_rows < 0", who);
  CBIS_REQUIRE(dtype == CBIS_F32 || dtype == CBIS_BF16, CBIS_ERR_UNSUPPORTED, "%s: dtype %d (fp32 or bf16)", who, dtype);
  if (n_rows == 0) return CBIS_OK;
  const int64_t width = (int64_t)c->n_kv_heads * c->head_dim;
  const size_t es = dtype == CBIS_F32 ? 4 : 2;
  CBIS_REQUIRE(K && V && page && offset, CBIS_ERR_INVALID, "%s: null pointer", who);
  CBIS_REQUIRE(ldk >= width && ldv >= width, CBIS_ERR_INVALID, "%s: row strides %lld, %lld below the row's %lld elements",
               who, (long long)ldk, (long long)ldv, (long long)width);
  CBIS_REQUIRE((((uintptr_t)K | (uintptr_t)V) & (es - 1)) == 0 && (((uintptr_t)page | (uintptr_t)offset) & 3u) == 0,
               CBIS_ERR_INVALID, "%s: misaligned pointer", who);
  a.n_rows = n_rows;
  a.k = K;
  a.v = V;
  a.ldk = ldk;
  a.ldv = ldv;
  a.page = page;
  a.offset = offset;
  a.parts = (int)cdiv(width, 64 * (16 / (int64_t)es));
  const int64_t grid = cdiv(n_rows, kTile) * a.parts;
  CBIS_REQUIRE(grid < (1LL << 31), CBIS_ERR_UNSUPPORTED, "%s: grid too large", who);
  if (dtype == CBIS_F32) rows_launch<float>(gather, a, (unsigned)grid, s);
  else rows_launch<uint16_t>(gather, a, (unsigned)grid, s);
  return check_launch(who);
}

constexpr int64_t kCUs = 256;

// Sizes that both the workspace queries and the launches go by.
struct Plan {
  int nsplit = 1, split_blocks = 1 << 24;
  int nh = 1, nhb = 1, tw = 1, waves = 1, groups = 1;  // decode
  int sw = 1, ncg = 1;   // chunk: staging items of a wave, column groups
  int64_t slots = 0;     // rows (or tile rows) of the partials
  size_t bytes = 0;
};

bool heads_ok(const cbis_kv8_attn_desc* d) {
  return d && geometry_ok(d->cache.n_kv_heads, d->cache.head_dim, d->cache.page_size) && d->n_heads > 0 &&
         d->n_heads % d->cache.n_kv_heads == 0;
}

int64_t table_tokens(const cbis_kv8_attn_desc* d) {
  return std::min<int64_t>(std::max<int64_t>(d->bt_stride, 0), (1 << 30) / d->cache.page_size) * d->cache.page_size;
}

// 64-token blocks of the longest row, as far as the host knows.
int64_t longest(const cbis_kv8_attn_desc* d) {
  int64_t tok = table_tokens(d);
  if (d->max_kv_len > 0) tok = std::min<int64_t>(tok, d->max_kv_len);
  return std::max<int64_t>(1, cdiv(tok, kBlk));
}

// Splits of `per` blocks, unless the caller names their tokens.
void set_splits(const cbis_kv8_attn_desc* d, int64_t blocks, int64_t per, Plan* p) {
  if (d->split_tokens > 0) per = d->split_tokens / kBlk;
  per = std::max<int64_t>(per, cdiv(blocks, 1 << 15));
  p->nsplit = (int)cdiv(blocks, per);
  p->split_blocks = (int)per;
  if (p->nsplit > 1) p->bytes = (size_t)p->slots * p->nsplit * d->n_heads * (d->cache.head_dim + 1) * 4;
}

Plan plan_decode(const cbis_kv8_attn_desc* d) {
  Plan p;
  const int group = d->n_heads / d->cache.n_kv_heads;
  if (group > 16) {
    p.nhb = d->cache.n_kv_heads * ((group + 15) / 16);
  } else {
    // kv heads of a workgroup: as many as make 128 dims, have columns and exist.
    p.nh = 128 / d->cache.head_dim;
    while (p.nh > 1 && (p.nh * group > 16 || p.nh / 2 >= d->cache.n_kv_heads)) p.nh /= 2;
    p.nhb = (d->cache.n_kv_heads + p.nh - 1) / p.nh;
  }
  p.slots = std::max(d->n_rows, 0);
  // The waves that share a row's head block: as many as bring the waves to
  // 4096, two rounds of what the GPU holds, so that rows of half the longest
  // one's length still fill it; no more than the blocks. us by waves, MI355X:
  //   192 rows of 256..4096 x 64 heads of 32                     1: 285  2: 277  4: 278  8: 312
  //   256 rows of 100 x 64 heads of 32 (4096)                    1: 29   2: 35   4: 49   8: 84
  //   64 rows of 1000 x 64 heads of 32 (1024)                    1: 48   2: 47   4: 50   8: 62
  //   61 rows of 500..16384, 32 / 8 heads of 128 (488)           1: 563  2: 319  4: 230  8: 193
  //   16 rows of 1000 x 64 heads of 32 (256)                     1: 37   2: 23   4: 16   8: 17
  // Past eight waves the keys are split over workgroups of eight, a CU's worth.
  // Up to 64 head blocks make one round of 256 workgroups, whose rows' lengths
  // matter little; more of them two rounds, since the rest of a GPU that is half
  // full is lost where the rows are uneven.  us by tokens of a split, equal rows /
  // rows of any length up to that (* what the rule takes):
  //   4 rows of 16384, 8 kv heads of 128   1024: 45 / 39  2048*: 35 / 31  4096: 50 / 43
  //   8 rows of 16384                      2048: 66 / 53  4096*: 57 / 50  8192: 86 / 73
  //   16 rows of 16384                     4096*: 109 / 79  8192: 100 / 84
  //   24 rows of 16384                     8192*: - / 93  16384: - / 134
  //   1 row of 4000, 64 heads of 32        256*: 12.4  512: 14.9  1024: 17  4096: 28
  // A row of 600 is faster whole (10.2; 256: 10.9), one of 1000 in splits (12.2; 11.0).
  const int64_t units = std::max<int64_t>(1, p.slots * p.nhb), blocks = longest(d);
  const int64_t part = d->split_tokens > 0 ? std::min<int64_t>(blocks, d->split_tokens / kBlk) : blocks;
  while (p.tw < kDecodeWaves && units * p.tw < 4096 && p.tw < part) p.tw *= 2;
  p.waves = std::max(p.tw, 4);
  p.groups = (int)cdiv(p.nhb, p.waves / p.tw);
  int64_t per = blocks;
  if (units <= 64 && blocks >= 16) per = std::max<int64_t>(cdiv(blocks, kCUs / units), 4);
  else if (units <= kCUs && blocks >= 16) per = std::max<int64_t>(cdiv(blocks, 2 * kCUs / units), 16);
  set_splits(d, blocks, per, &p);
  return p;
}

Plan plan_chunk(const cbis_kv8_attn_desc* d, int n_tiles) {
  Plan p;
  const int group = d->n_heads / d->cache.n_kv_heads;
  p.slots = (int64_t)std::max(n_tiles, 0) * CBIS_PREFILL_TILE_ROWS;
  const int64_t blocks = longest(d);
  if (d->cache.head_dim == 32) {
    p.ncg = (CBIS_PREFILL_TILE_ROWS * group + kChunkCols - 1) / kChunkCols;
    const int64_t units = std::max<int64_t>(1, (int64_t)n_tiles * d->cache.n_kv_heads * p.ncg);
    const int64_t part = d->split_tokens > 0 ? std::min<int64_t>(blocks, d->split_tokens / kBlk) : blocks;
    // Waves that share the keys of 32 columns: as many as bring the waves to 2048,
    // two to a SIMD.  us by that goal, 64 heads of 32, MI355X:
    //   two chunks of 512, 0 and 512 cached      1: 23.7  2048: 23.5  4096: 23.2  8192: 27.9
    //   512 rows after 16384                     1: 224   2048: 192   4096: 201   8192: 220
    //   512 fresh rows                           1: 12.5  2048: 10.8  4096: 13.8  8192: 21.6
    //   16 rows after 32000                      1: 118   2048: 61    4096: 61    8192: 61
    // But 8 only where that is no more than a workgroup per CU, which does not hold
    // two (of four it holds three): 3 x 64 rows after 1000 18.6 with 8, 14.7 with 4, 3 x
    // 20 after 5000 40 and 31.
    while (p.tw < (units <= kCUs ? 8 : 4) && units * p.tw < 2048 && p.tw < part) p.tw *= 2;
    p.waves = std::max(p.tw, 4);
    // Splits for what the CUs hold at once, from 48 blocks on.  us by tokens of
    // a split (* the rule's): 64 rows of 64 heads after 2000  1024: 19  2048*: 14,
    // after 4000  1024: 22  2048*: 18  4096: 20, after 32000  8192: 64  16384*: 60
    // 32768: 93; 64 rows of 8 heads after 4000  256*: 11.4  1024: 14  4096: 19.
    const int64_t room = units <= kCUs ? kCUs : 3 * kCUs;
    if (blocks >= 48) set_splits(d, blocks, std::max<int64_t>(cdiv(blocks, std::max<int64_t>(1, room / units)), 4), &p);
    else set_splits(d, blocks, blocks, &p);
    return p;
  }
  // As many waves as a kv head's columns fill, times the parts of the keys: up to 8,
  // or 4 where the longest row has no more than 32 blocks: smaller pieces, two to a
  // CU, even out the tiles' lengths, but each converts K and V for itself.  us with
  // 8 / 4 waves:
  //   32 / 8 heads of 128  512 fresh rows 27 / 23  64 after 1000 20 / 19  1500 after 300 69 / 63
  //     512 after 4096 67 / 80  4 x 512 after 8192 298 / 324  8192 fresh rows 571 / 584
  //   16 / 4 heads of 64   512 fresh rows 13.8 / 12.1  512 after 4096 31 / 38
  // Two parts of q of 128 dims leave a CU no room for a second workgroup (8 x 300
  // rows after 200 53 / 62, 512 fresh ones 30 / 24).
  const int KG = 128 / d->cache.head_dim;
  const int cols = chunk_cols(d->cache.head_dim, d->out_dtype == CBIS_F32 ? 3 : 1);
  const int want = (CBIS_PREFILL_TILE_ROWS * group + cols - 1) / cols;
  const bool alone = KG == 1 && d->q_dtype == CBIS_F32 && d->out_dtype == CBIS_BF16;
  const int64_t eights = (int64_t)n_tiles * d->cache.n_kv_heads * cdiv(want, 8 / KG);
  if (blocks <= 32 && (!alone || eights <= kCUs / 2)) p.sw = 2;
  while (p.sw < 4 / KG && 4 / p.sw >= want * KG) p.sw *= 2;
  const int wh = 8 / p.sw / KG;
  p.ncg = (want + wh - 1) / wh;
  const int64_t units = std::max<int64_t>(1, (int64_t)n_tiles * d->cache.n_kv_heads * p.ncg);
  // Splits for one workgroup per CU, of at least sqrt(blocks) / 2 blocks: more of
  // them cost more to join than they save.  us by tokens of a split (* the rule's):
  //   32 / 8 heads of 128, 512 rows after 16384  4 splits* 174, 8 175 and another 9 us of joining
  //     64 rows after 300    64: 15.6  128*: 17  512: 21     after 1000  64: 21  128*: 20  256: 22  512: 29
  //     64 rows after 4096   128: 37  256*: 28  512: 33      256 rows after 500  64: 36  128*: 25  512: 33
  //   16 / 4 heads of 64, 64 rows after 4096  128: 22  256*: 17  512: 19   after 300  128: 12.4  whole*: 11.9
  int64_t per = blocks;
  if (blocks > 4 * KG) {
    per = KG;
    while (4 * per * per < blocks) per += KG;
    per = std::max<int64_t>({per, 2, cdiv(blocks, std::max<int64_t>(1, kCUs / units))});
    // A CU holds two of the smaller workgroups: where keys are long, splits for both
    // (32 heads of 64: 512 rows after 16384 185 -> 146, 3 x 28 after 12149 75 -> 62).
    if (p.sw > 1 && per > 48) per = std::max<int64_t>(48, cdiv(blocks, std::max<int64_t>(1, 2 * kCUs / units)));
  }
  set_splits(d, blocks, per, &p);
  return p;
}

int attn_args(const cbis_kv8_attn_desc* d, AttnArgs* a, const char* who) {
  CBIS_REQUIRE(d, CBIS_ERR_INVALID, "%s: null descriptor", who);
  const int rc = make_pages(&d->cache, &a->c, who);
  if (rc) return rc;
  CBIS_REQUIRE(d->n_heads > 0 && d->n_heads % d->cache.n_kv_heads == 0, CBIS_ERR_INVALID,
               "%s: n_heads %d must be a multiple of n_kv_heads %d", who, d->n_heads, d->cache.n_kv_heads);
  CBIS_REQUIRE((d->q_dtype == CBIS_F32 || d->q_dtype == CBIS_BF16) && (d->out_dtype == CBIS_F32 || d->out_dtype == CBIS_BF16),
               CBIS_ERR_UNSUPPORTED, "%s: q dtype %d, out dtype %d (fp32 or bf16)", who, d->q_dtype, d->out_dtype);
  CBIS_REQUIRE(d->split_tokens >= 0 && d->split_tokens % kBlk == 0, CBIS_ERR_INVALID,
               "%s: split_tokens %d must be a multiple of %d, or 0", who, d->split_tokens, kBlk);
  CBIS_REQUIRE(d->max_kv_len >= 0, CBIS_ERR_INVALID, "%s: max_kv_len < 0", who);
  const int64_t width = (int64_t)d->n_heads * d->cache.head_dim;
  CBIS_REQUIRE(d->q && d->out && d->block_table, CBIS_ERR_INVALID, "%s: null pointer", who);
  CBIS_REQUIRE(d->ldq >= width && d->ldo >= width && d->bt_stride > 0, CBIS_ERR_INVALID,
               "%s: row strides %lld, %lld below the row's %lld elements, or bt_stride %lld", who, (long long)d->ldq,
               (long long)d->ldo, (long long)width, (long long)d->bt_stride);
  const size_t qs = d->q_dtype == CBIS_F32 ? 4 : 2, os = d->out_dtype == CBIS_F32 ? 4 : 2;
  CBIS_REQUIRE(((uintptr_t)d->q & (qs - 1)) == 0 && ((uintptr_t)d->out & (os - 1)) == 0 &&
                   (((uintptr_t)d->block_table | (uintptr_t)d->rows | (uintptr_t)d->row_bt | (uintptr_t)d->row_pos) & 3u) == 0,
               CBIS_ERR_INVALID, "%s: misaligned pointer", who);
  a->n_heads = d->n_heads;
  a->group = d->n_heads / d->cache.n_kv_heads;
  a->q = d->q;
  a->ldq = d->ldq;
  a->q_bf16 = d->q_dtype == CBIS_BF16;
  a->q_vec = (((uintptr_t)d->q | (uintptr_t)(d->ldq * qs)) & 15u) == 0;
  a->bt = d->block_table;
  a->bt_stride = d->bt_stride;
  a->out = d->out;
  a->ldo = d->ldo;
  a->out_bf16 = d->out_dtype == CBIS_BF16;
  a->out_vec = (((uintptr_t)d->out | (uintptr_t)(d->ldo * os)) & (4 * os - 1)) == 0;
  a->max_tok = (int)table_tokens(d);
  a->qscale = kLog2e / sqrtf((float)d->cache.head_dim);
  return CBIS_OK;
}

int take_workspace(const cbis_kv8_attn_desc* d, const Plan& p, AttnArgs* a, const char* who) {
  a->nsplit = p.nsplit;
  a->split_blocks = p.split_blocks;
  if (p.nsplit == 1) return CBIS_OK;
  CBIS_REQUIRE(d->workspace && d->workspace_bytes >= p.bytes, CBIS_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", who, p.bytes, d->workspace ? d->workspace_bytes : (size_t)0);
  CBIS_REQUIRE(((uintptr_t)d->workspace & 15u) == 0, CBIS_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
  a->part = (float*)d->workspace;
  a->lse = a->part + p.slots * p.nsplit * d->n_heads * d->cache.head_dim;
  return CBIS_OK;
}

int merge(const AttnArgs& a, const Plan& p, hipStream_t s, const char* who) {
  int share = 1;  // one group per two splits, as far as the wave has them
  while (share * 2 <= 256 / a.c.head_dim && share * 2 < p.nsplit) share *= 2;
  const int64_t grid = cdiv(p.slots * a.n_heads * (a.c.head_dim / 4) * share, 256);
  CBIS_REQUIRE(grid < (1LL << 31), CBIS_ERR_UNSUPPORTED, "%s: grid too large", who);
  if (a.c.head_dim == 32) kv8_merge_kernel<32><<<(unsigned)grid, 256, 0, s>>>(a, p.slots, share);
  else if (a.c.head_dim == 64) kv8_merge_kernel<64><<<(unsigned)grid, 256, 0, s>>>(a, p.slots, share);
  else kv8_merge_kernel<128><<<(unsigned)grid, 256, 0, s>>>(a, p.slots, share);
  return check_launch(who);
}

template <int HD, int QP, int PP>
void decode_heads(const AttnArgs& a, const Plan& p, unsigned grid, hipStream_t s) {
  const int threads = p.waves * 64;
  const size_t lds = p.tw > 1 ? (size_t)p.waves * 16 * (HD + 5) * sizeof(float) : 0;
  if constexpr (HD <= 32) {
    if (p.nh == 4) return kv8_decode_kernel<HD, 4, QP, PP><<<grid, threads, lds, s>>>(a);
  }
  if constexpr (HD <= 64) {
    if (p.nh == 2) return kv8_decode_kernel<HD, 2, QP, PP><<<grid, threads, lds, s>>>(a);
  }
  kv8_decode_kernel<HD, 1, QP, PP><<<grid, threads, lds, s>>>(a);
}

template <int QP, int PP>
void decode_parts(const AttnArgs& a, const Plan& p, unsigned grid, hipStream_t s) {
  if (a.c.head_dim == 32) decode_heads<32, QP, PP>(a, p, grid, s);
  else if (a.c.head_dim == 64) decode_heads<64, QP, PP>(a, p, grid, s);
  else decode_heads<128, QP, PP>(a, p, grid, s);
}

template <int HD, int QP, int PP>
void chunk_heads(const AttnArgs& a, const Plan& p, unsigned grid, hipStream_t s) {
  const size_t lds = chunk_lds<HD>(8 / p.sw);
  if constexpr (HD == 128) {
    if (p.sw == 4) return kv8_chunk_kernel<HD, 4, QP, PP><<<grid, 128, lds, s>>>(a);
  }
  if constexpr (HD >= 64) {
    if (p.sw == 2) return kv8_chunk_kernel<HD, 2, QP, PP><<<grid, 256, lds, s>>>(a);
  }
  kv8_chunk_kernel<HD, 1, QP, PP><<<grid, 512, lds, s>>>(a);
}

template <int QP, int PP>
void chunk_parts(const AttnArgs& a, const Plan& p, unsigned grid, hipStream_t s) {
  if (a.c.head_dim == 32) {
    const size_t join = p.tw > 1 ? (size_t)p.waves * kChunkCols * (32 + 5) * sizeof(float) : 0;
    kv8_chunk32_kernel<QP, PP><<<grid, p.waves * 64, std::max(join, (size_t)p.waves * 64 * sizeof(_Float16)), s>>>(a);
  } else if (a.c.head_dim == 64) {
    chunk_heads<64, QP, PP>(a, p, grid, s);
  } else {
    chunk_heads<128, QP, PP>(a, p, grid, s);
  }
}

}  // namespace
}  // namespace cbis

using namespace cbis;

extern "C" {

size_t cbis_kv8_page_bytes(int n_kv_heads, int head_dim, int page_size) {
  if (!geometry_ok(n_kv_heads, head_dim, page_size)) return 0;
  return (size_t)page_size * n_kv_heads * (head_dim + 1);
}

int cbis_kv8_scatter(const cbis_kv8_cache* c, int n_rows, int src_dtype, const void* K, int64_t ldk, const void* V,
                     int64_t ldv, const int* write_page, const int* write_offset, cbis_stream_t stream) {
  return kv8_rows(false, c, n_rows, src_dtype, K, ldk, V, ldv, write_page, write_offset, (hipStream_t)stream,
                  "cbis_kv8_scatter");
}

int cbis_kv8_gather(const cbis_kv8_cache* c, int n_rows, int dst_dtype, void* K, int64_t ldk, void* V, int64_t ldv,
                    const int* read_page, const int* read_offset, cbis_stream_t stream) {
  return kv8_rows(true, c, n_rows, dst_dtype, K, ldk, V, ldv, read_page, read_offset, (hipStream_t)stream,
                  "cbis_kv8_gather");
}

size_t cbis_kv8_attention_workspace_size(const cbis_kv8_attn_desc* d) { return heads_ok(d) ? plan_decode(d).bytes : 0; }

int cbis_kv8_attention(const cbis_kv8_attn_desc* d, cbis_stream_t stream) {
  const char* who = "cbis_kv8_attention";
  AttnArgs a = {};
  int rc = attn_args(d, &a, who);
  if (rc) return rc;
  CBIS_REQUIRE(d->n_rows >= 0, CBIS_ERR_INVALID, "%s: n_rows < 0", who);
  if (d->n_rows == 0) return CBIS_OK;
  CBIS_REQUIRE(d->row_pos, CBIS_ERR_INVALID, "%s: null row_pos", who);
  const Plan p = plan_decode(d);
  if ((rc = take_workspace(d, p, &a, who))) return rc;
  a.n_rows = d->n_rows;
  a.rows = d->rows;
  a.row_bt = d->row_bt;
  a.row_pos = d->row_pos;
  a.nhb = p.nhb;
  a.tw = p.tw;
  const int64_t grid = p.slots * p.groups * p.nsplit;
  CBIS_REQUIRE(grid < (1LL << 31), CBIS_ERR_UNSUPPORTED, "%s: grid too large", who);
  hipStream_t s = (hipStream_t)stream;
  if (a.out_bf16) {
    if (a.q_bf16) decode_parts<1, 1>(a, p, (unsigned)grid, s);
    else decode_parts<2, 1>(a, p, (unsigned)grid, s);
  } else {
    decode_parts<3, 2>(a, p, (unsigned)grid, s);  // bf16 q: its second and third parts are zero
  }
  rc = check_launch(who);
  return rc || p.nsplit == 1 ? rc : merge(a, p, s, who);
}

size_t cbis_kv8_chunk_attention_workspace_size(const cbis_kv8_attn_desc* d, int n_tiles) {
  return heads_ok(d) ? plan_chunk(d, n_tiles).bytes : 0;
}

int cbis_kv8_chunk_attention(const cbis_kv8_attn_desc* d, int n_tiles, const int* tiles, cbis_stream_t stream) {
  const char* who = "cbis_kv8_chunk_attention";
  AttnArgs a = {};
  int rc = attn_args(d, &a, who);
  if (rc) return rc;
  CBIS_REQUIRE(n_tiles >= 0, CBIS_ERR_INVALID, "%s: n_tiles < 0", who);
  if (n_tiles == 0) return CBIS_OK;
  CBIS_REQUIRE(tiles && ((uintptr_t)tiles & 15u) == 0, CBIS_ERR_INVALID,
               "%s: tiles must be a 16-byte aligned device array [n_tiles][4]", who);
  const Plan p = plan_chunk(d, n_tiles);
  if ((rc = take_workspace(d, p, &a, who))) return rc;
  a.tiles = tiles;
  a.n_tiles = n_tiles;
  a.ncg = p.ncg;
  a.tw = p.tw;
  const int64_t units = (int64_t)n_tiles * p.nsplit * d->cache.n_kv_heads * p.ncg;
  const int64_t grid = d->cache.head_dim == 32 ? cdiv(units, p.waves / p.tw) : units;
  CBIS_REQUIRE(grid < (1LL << 31), CBIS_ERR_UNSUPPORTED, "%s: grid too large", who);
  hipStream_t s = (hipStream_t)stream;
  if (a.out_bf16) {
    if (a.q_bf16) chunk_parts<1, 1>(a, p, (unsigned)grid, s);
    else chunk_parts<2, 1>(a, p, (unsigned)grid, s);
  } else {
    chunk_parts<3, 2>(a, p, (unsigned)grid, s);
  }
  rc = check_launch(who);
  return rc || p.nsplit == 1 ? rc : merge(a, p, s, who);
}

}  // extern "C"
