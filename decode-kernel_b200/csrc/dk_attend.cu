// dk_attend.cu -- attention of a step's queries over a paged cache held in 8
// bits (int8 or e4m3) with one fp32 scale per page and KV head.
//
// For a query row q of KV head h and the cached tokens j its mask leaves,
//   s_j = scale * ks[page(j)] * (q . Kcode_j)         out = sum_j p_j V_j
//   p_j = exp(s_j) / sum_i exp(s_i)                   V_j = vs[page(j)] * Vcode_j
// computed in one pass with a running maximum.  The page's V scale goes into
// the exponent: with t_j = s_j log2(e) + log2(vs_j) and w_j = 2^(t_j - m),
//   out = (sum_j w_j Vcode_j) / (sum_j w_j / vs_j),
// so the codes enter the tensor core unscaled (int8 and e4m3 are exact in
// fp16) and w_j is at most 2^15, whatever the scales.  w_j is rounded to fp16
// (11 bits; a relative 2^-12 on each weight, the size of the rounding of an
// fp16 output); scores, maxima, sums and outputs are fp32.  m puts the largest
// weight at 2^7 or above, so that weights keep their 11 bits down to 2^-21 of it
// and something down to 2^-32 (with the largest at 1, a token of large score and
// little V would wipe out all that come to 2^-25 of it, in any number).
//
// What bounds it: the cache's bytes from HBM, up to about 16 query rows per KV
// head; beyond, the matrix instructions.  A tile of 16 tokens and 8 query rows
// takes 16 m16n8k16 instructions for heads of 128, in which the tokens (then
// the channels) are the 16 rows and the query rows the 8 columns, so no row is
// padding when 8 query heads share a KV head.  (tcgen05 would take the same
// arrangement, 128 tokens by 16 to 256 query rows, but with the codes converted
// and stored to shared or tensor memory once more, as fp16; for the rows past 16
// that is not measured.)
//   K: lane (g, c) takes tokens g and g + 8, channels 32c..32c+31: word s of a
//      row is its part of the s-th k step (the sum over channels may run in any
//      order, so q is loaded in the same one).
//   V: lane (g, c) takes tokens 2c, 2c+1, 2c+8, 2c+9, channels 16g..16g+15: byte
//      pairs of two tokens are interleaved with PRMT and converted.
//   P: the score tile is [token][row]; movmatrix transposes it into the second
//      product's operand.
// The codes reach shared memory by asynchronous 16-byte copies, in whole
// 128-byte lines, into a ring that each warp has for itself: no barrier but
// the warp's own, and the copies of a warp's next units are under way while one
// is added up, across the segments' borders too.  (Straight from global memory
// to the fragments' registers the same cases take 1.1 to 1.2 times as long: one
// unit ahead is all that the registers hold, and the addresses spill.)
//
// Split: the units of all (request, KV head, row tile) segments form one line,
// which the CTAs share evenly, and each CTA's warps share its part evenly, so
// the split follows the lengths as they are on the device; no host sync and no
// padding to the longest.  A segment that a warp covers alone is written at
// once; the other parts meet in shared memory, and a segment that several CTAs
// share is joined by whichever of them arrives last, always in the same order
// of parts.
//
// Measured on one B200 (6550 GB/s copied): four contexts of 131 thousand tokens,
// 64 query heads over 8 of 128, e4m3: 167 us, 6.2 TB/s; 32 requests of 0 to 8192
// tokens, 32 over 8 heads, int8: 56 us, 5.0 TB/s, of which 40 us stream and the
// rest is the call's start, the slowest warps and the joins; 200 requests of up
// to 1900 tokens, a window of 1000, 12 heads of 64, e4m3: 52 us, 4.4 TB/s; 17
// requests of five queries (20 rows a KV head), 0.8 to 4 thousand tokens: 36 us;
// one request of 700 tokens 11.1 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dk_device.cuh"
#include "dk_host.h"

namespace dk {
namespace {

constexpr int kTile = 16;             // tokens of a tile: of one page, one matrix instruction's rows
constexpr int kMaxRequests = 1024;    // requests of one launch (their prefix sums are in shared memory)
constexpr int kShort = 96;            // tiles of segments that no two CTAs share, where there are many
constexpr int kVeryShort = 36;        // places of segments that no two CTAs share, however few
constexpr float kFarBelow = -1e30f;   // maximum of a row that has seen no token
constexpr float kTop = 7.f;           // log2 of the largest weight where a row's maximum is up to date
constexpr float kSlack = 8.f;         // it may lag its scores by this much (log2)
constexpr float kLeastScale = 8.4703294725430034e-22f;  // 2^-70: keeps sum w / vs finite

struct AttendArgs {
  const void* q;
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scale;
  const float* v_scale;
  const int* table;
  const int* lengths;
  const int* starts;
  void* out;
  float* lse;
  void* workspace;
  int* counters;
  float* partials;
  float* early;
  long long q_token_stride, q_head_stride;
  long long k_head_stride, v_head_stride;
  uint32_t k_block_stride, k_token_stride, v_block_stride, v_token_stride;
  int table_stride, max_blocks, blocks, block_size, tiles_per_block;
  int requests, tokens, kv_heads, group;
  int heads;                          // KV heads of the launch, from the pointers' on
  unsigned group_magic, block_magic;  // for over()
  float scale_log2;
  int causal, window, bf16;
};

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Four codes of one word to two half2: (b0, b1) and (b2, b3).
template <bool E4M3>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (E4M3) {
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n"
        " cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // code + 128 in the mantissa of 1024: 1152 + code, exact, less 1152.
    const uint32_t u = w ^ 0x80808080u;
    lo = hsub2_u32(prmt(u, 0x64646464u, 0x4140), 0x64806480u);
    hi = hsub2_u32(prmt(u, 0x64646464u, 0x4342), 0x64806480u);
  }
}

// The kernel may start while the call before it still runs (programmatic
// launch), so nothing is read through the non-coherent path: that data would
// have to be constant for the kernel's whole life.
__device__ __forceinline__ int ld_int(const int* p) {
  int x;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(x) : "l"(p));
  return x;
}

__device__ __forceinline__ uint4 ld_quad(const void* p) {
  uint4 r;
  asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

// Asynchronous copies into shared memory: 16 bytes past L1, or 4.
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

template <int WORDS>
__device__ __forceinline__ void lds_words(uint32_t at, uint32_t* r) {
  if constexpr (WORDS == 4) {
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
  } else {
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(at));
  }
}

// x / by for 0 <= x < 2^31, with magic = ceil(2^32 / by) (0 for by = 1).
__device__ __forceinline__ int over(int x, int by, unsigned magic) {
  if (magic == 0) return x;
  const int q = __umulhi(x, magic);  // the quotient or one more
  return q - ((long long)q * by > x);
}

// One (request, KV head, row tile): where its rows, tokens and units are.
struct Segment {
  int request, head, tile;
  int length, fresh, first_token;  // tokens held, queries, row of the first query in q
  int which, all;                  // its number among the request's segments, and how many they are
  int unit0, units;                // its first unit among the request's, and how many
  int begin;                       // place of its first unit in the line of all units
  int blocks;                      // pages of its request
};

// PACKED: the tokens of a page's head are neighbours in memory, so the rows of
// a unit lie at fixed offsets.
// MT: tiles of a unit, which a warp adds up side by side.
template <int D, int NT, int MT, bool E4M3, bool PACKED, int W, int S>
struct Attend {
  static constexpr int kRows = 8 * NT;
  static constexpr int kKWords = D / 16;  // words of a lane's part of a K row
  static constexpr int kVWords = D / 32;  // words of a lane's part of a V row
  static constexpr int kSlots = 2 * W;    // a warp's parts of segments: an early one and its last
  // Places in the line that a segment's start counts for: its queries' latency
  // and its rows' end take as long as this many units.
  static constexpr int kStart = NT >= 3 ? 2 : 1;
  static constexpr int kUnit = MT * kTile;  // tokens of a unit
  // A stage: each tile's K and V, and their scales.  Multiples of 128 bytes, so
  // that the places of pieces differ by an exclusive or of their low bits.
  static constexpr int kTileBytes = 2 * kTile * D, kScales = MT * kTileBytes;
  static constexpr int kStage = kScales + 128;
  // The queries' operands stay in registers while those hold them beside the
  // output's; from 24 rows of 128 on they are read from shared memory.
  static constexpr bool kQShared = NT * D > 256;
  static constexpr int kQBytes = kQShared ? NT * kKWords * 256 : 0;
  static constexpr int kWarp = S * kStage + kQBytes;  // a warp's shared memory
  static_assert(kRows * D * 4 <= kWarp, "a part fits it");

  struct Shared {
    unsigned char ring[W][kWarp];  // stages and queries; at the end the warp's last part: float [kRows][D]
    float m[kSlots][kRows];
    float l[kSlots][kRows];
    // Of the joins: a used slot's part and factors, a group's first part and the
    // places of its rows.
    const float* part[kSlots];
    float factor[kSlots][kRows];
    float by[kSlots][kRows];
    int place[kSlots][kRows];
    int group[kSlots + 1];
    Segment seg[kSlots];
    Segment fed[W], now[W];            // the segments whose units a warp copies and adds up
    int4 rows[W][kRows];               // of the latter's rows: token (-1: no such row), head, low, high
    int used[kSlots];
    int last[2];
    int total[W], longest[W], segments[W];
    int range[2];
  };

  // Place of 16-byte piece p of a unit's row: the pieces that eight lanes read
  // together, of K (two rows) and of V (four rows two apart), lie in different
  // banks.
  __device__ static __forceinline__ int place(int row, int p) {
    if constexpr (D == 64) {
      const int line = row >> 1;
      return line * 128 + (((row & 1) * 4 + p) ^ ((line & 3) * 2)) * 16;
    } else if constexpr (D == 128) {
      return row * D + (p ^ (row & 7)) * 16;
    } else {
      return row * D + (p ^ (((row ^ (row >> 1)) & 1) | (row & 4))) * 16;
    }
  }
  // A lane's places, of which the others follow by offsets and exclusive ors:
  // place(row + j * kStep, p) = (place(row, p) ^ copy_turn(j)) + j * 512,
  static constexpr int kPieces = D / 16, kStep = 512 / D;  // pieces of a row, rows of a warp's copy
  __device__ static constexpr int copy_turn(int j) { return D == 64 ? 0 : D == 128 ? (j & 1) * 64 : (j & 1) * 16 + (j & 2) * 32; }
  // place(g, 2c + 1) = place(g, 2c) ^ 16, place(2c + 1, p) = (place(2c, p) ^ kOdd) + kOddRow.
  static constexpr int kOdd = D == 64 ? 64 : 16, kOddRow = D == 64 ? 0 : D;

  // The first token that query i of a request sees with a window.  The maximum
  // inside keeps the sum within 32 bits for any window and more queries than tokens.
  __device__ static __forceinline__ int window_from(const AttendArgs& a, int length, int fresh, int i) {
    return max(0, max(0, length - a.window) - (fresh - 1 - i));
  }
  __device__ static __forceinline__ int units_of(const AttendArgs& a, int length, int fresh, int& unit0) {
    unit0 = 0;
    if (a.window > 0) unit0 = window_from(a, length, fresh, 0) / kUnit;
    return max(1, (length + kUnit - 1) / kUnit - unit0);
  }
  // Row tiles of a request: of those of its queries that the call has rows for.
  __device__ static __forceinline__ int tiles_of(const AttendArgs& a, int first, int fresh) {
    return (min(fresh, max(0, a.tokens - max(0, first))) * a.group + kRows - 1) / kRows;
  }
  // The requests' numbers in shared memory: prefix[r] = the place of request
  // r's first unit in the line (one more entry than requests), then the tokens
  // that each holds, and if there are starts those (again one more).
  __device__ static __forceinline__ void request_of(const AttendArgs& a, const int* prefix, int r, int& length, int& fresh, int& first) {
    const int* lengths = prefix + a.requests + 1;
    length = lengths[r];
    if (a.starts) {
      const int* starts = lengths + a.requests;
      first = starts[r];
      fresh = max(0, starts[r + 1] - first);
    } else {
      first = r;
      fresh = 1;
    }
  }

  // Segment `which` of request r.
  __device__ static __forceinline__ Segment segment_of(const AttendArgs& a, const int* prefix, int r, int which) {
    Segment s;
    s.request = r;
    request_of(a, prefix, r, s.length, s.fresh, s.first_token);
    s.units = units_of(a, s.length, s.fresh, s.unit0);
    s.which = which;
    s.begin = prefix[r] + which * (s.units + kStart) + kStart;
    s.blocks = over((s.length + kTile - 1) / kTile + a.tiles_per_block - 1, a.tiles_per_block, a.block_magic);
    const int tiles = tiles_of(a, s.first_token, s.fresh);
    s.all = tiles * a.heads;
    s.head = tiles == 1 ? which : which / tiles;
    s.tile = which - s.head * tiles;
    return s;
  }
  // The segment of place u of the line.
  __device__ static __forceinline__ Segment segment_at(const AttendArgs& a, const int* prefix, int u) {
    // The last request whose first unit is at or before u, 32 candidates at a time.
    const int lane = threadIdx.x & 31;
    int lo = 0;
    for (int n = a.requests; n > 1;) {
      const int step = (n + 31) >> 5, at = lane * step;
      const uint32_t before = __ballot_sync(0xffffffffu, at < n && prefix[lo + at] <= u);
      const int skip = (31 - __clz(before | 1u)) * step;
      lo += skip;
      n = min(step, n - skip);
    }
    Segment s = segment_of(a, prefix, lo, 0);
    const int which = (u - (s.begin - kStart)) / (s.units + kStart);
    return which ? segment_of(a, prefix, lo, which) : s;
  }
  // The segment after segment `which` of request r, which ends before place u.
  __device__ static __forceinline__ void after(const AttendArgs& a, const int* prefix, int r, int which, int u, int& next_r, int& next_which) {
    next_r = r;
    next_which = which + 1;
    if (u < prefix[r + 1]) return;
    next_which = 0;
    ++next_r;  // some request after r has units
    while (next_r + 1 < a.requests && prefix[next_r + 1] <= u) ++next_r;
  }

  // Token range [low, high) that query row `row` of the segment sees, and its
  // place in q and out; false where the tile has no such row.
  __device__ static __forceinline__ bool row_of(const AttendArgs& a, const Segment& s, int row, int& token, int& head, int& low, int& high) {
    const int all = s.tile * kRows + row;
    const int i = over(all, a.group, a.group_magic);
    token = s.first_token + i;
    head = s.head * a.group + all - i * a.group;
    low = high = 0;
    if (i >= s.fresh || (unsigned)token >= (unsigned)a.tokens) return false;
    high = a.causal ? min(s.length, max(0, s.length - s.fresh + i + 1)) : s.length;
    if (a.window > 0) low = window_from(a, s.length, s.fresh, i);
    return true;
  }

  // A row of q as this lane's words of the B operand, in K's order of channels.
  __device__ static __forceinline__ void load_q(const AttendArgs& a, const int4& row, uint32_t (&b)[2 * kKWords]) {
    const int c = threadIdx.x & 3;
    constexpr int kSpan = D >= 128 ? 32 : 16;  // channels of a lane's contiguous piece
#pragma unroll
    for (int i = 0; i < 2 * kKWords; ++i) b[i] = 0;
    if (row.x >= 0) {
      const uint16_t* p = static_cast<const uint16_t*>(a.q) + row.x * a.q_token_stride + row.y * a.q_head_stride + c * kSpan;
#pragma unroll
      for (int i = 0; i < kKWords / 2; ++i) {  // 8 channels each
        const int at = (i * 8) % kSpan + (i * 8) / kSpan * 128;
        const uint4 x = ld_quad(p + at);
        b[4 * i] = x.x; b[4 * i + 1] = x.y; b[4 * i + 2] = x.z; b[4 * i + 3] = x.w;
      }
    }
  }
  // bf16 rows to fp16: scaled by a power of two, which the return value undoes,
  // to 2^14 and above, so that values keep their 8 bits down to 2^-31 of the row's
  // largest (and 2^-39 of it is still not 0).
  __device__ static __forceinline__ float convert_q(const AttendArgs& a, uint32_t (&b)[2 * kKWords]) {
    if (!a.bf16) return 1.f;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * kKWords; ++i)
      top = fmaxf(top, fmaxf(fabsf(__uint_as_float(b[i] << 16)), fabsf(__uint_as_float(b[i] & 0xffff0000u))));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^(14 - e) with e the exponent of the row's largest value, within fp32's range.
    const int e = min(max((int)(__float_as_uint(top) >> 23), 15), 254);
    const float down = __uint_as_float((uint32_t)(254 + 14 - e) << 23), up = __uint_as_float((uint32_t)(e - 14) << 23);
#pragma unroll
    for (int i = 0; i < 2 * kKWords; ++i)
      b[i] = pack_half2(__uint_as_float(b[i] << 16) * down, __uint_as_float(b[i] & 0xffff0000u) * down);
    return up;
  }

  __device__ static __forceinline__ void store_row(const AttendArgs& a, long long at, const float4& x) {
    uint2 w;
    if (a.bf16) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(x.x, x.y), r = __floats2bfloat162_rn(x.z, x.w);
      w.x = *reinterpret_cast<const uint32_t*>(&p);
      w.y = *reinterpret_cast<const uint32_t*>(&r);
    } else {
      w.x = pack_half2(x.x, x.y);
      w.y = pack_half2(x.z, x.w);
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = w;
  }

  // The warp's copies: its units in their order, across segments, each into
  // the next stage of its ring.
  struct Feed {
    const uint8_t* k;  // the lane's first piece in page 0 of the segment's head
    const uint8_t* v;
    const float* scale;  // of K (even lanes) or V there
    uint32_t to;         // the lane's place in the next stage
    int unit, end, segment_end;  // place of the next unit in the line, the warp's end, the segment's
    int block, sub, page, next_page;
    uint32_t hidden;  // of each stage's tiles (bits): the page is outside the pool

    __device__ __forceinline__ int page_at(const AttendArgs& a, const Segment& s, int b) const {
      return b < s.blocks ? ld_int(a.table + (long long)s.request * a.table_stride + b) : -1;
    }

    // From here units of segment s.
    __device__ __forceinline__ void enter(const AttendArgs& a, const Segment& s) {
      const int lane = threadIdx.x & 31;
      const int row = lane / kPieces, piece = lane % kPieces;
      segment_end = s.begin + s.units;
      k = a.k + s.head * a.k_head_stride + (PACKED ? row * D : row * (long long)a.k_token_stride) + piece * 16;
      v = a.v + s.head * a.v_head_stride + (PACKED ? row * D : row * (long long)a.v_token_stride) + piece * 16;
      scale = (lane & 1 ? a.v_scale : a.k_scale) + s.head;
      unit = max(unit, s.begin);
      const int t = (s.unit0 + unit - s.begin) * MT;
      block = over(t, a.tiles_per_block, a.block_magic);
      sub = t - block * a.tiles_per_block;
      page = page_at(a, s, block);
      next_page = page_at(a, s, block + 1);
    }

    // Copies the next unit, if there is one, into stage `at` (its number,
    // `stage`); always one group.
    __device__ __forceinline__ void next(const AttendArgs& a, const int* prefix, Segment& s, int offset, int stage) {
      if (unit == segment_end && unit < end) {
          int r, which;
        after(a, prefix, s.request, s.which, segment_end, r, which);
        __syncwarp();  // every lane has read s
        const Segment t = segment_of(a, prefix, r, which);
        if ((threadIdx.x & 31) == 0) s = t;
        __syncwarp();
        enter(a, t);
      }
      if (unit < end) {
        const int lane = threadIdx.x & 31;
        const uint32_t scales = to - place(lane / kPieces, lane % kPieces) + offset + kScales + lane * 4;
#pragma unroll
        for (int h = 0; h < MT; ++h) {
          const bool good = (unsigned)page < (unsigned)a.blocks;
          const uint32_t p = good ? page : 0, bit = stage * MT + h;
          hidden = (hidden & ~(1u << bit)) | ((good ? 0u : 1u) << bit);
          const uint32_t first = sub * kTile;
          const uint8_t* from_k = k + (uint64_t)p * a.k_block_stride + (PACKED ? first * D : first * a.k_token_stride);
          const uint8_t* from_v = v + (uint64_t)p * a.v_block_stride + (PACKED ? first * D : first * a.v_token_stride);
          const uint32_t at = to + offset + h * kTileBytes;
#pragma unroll
          for (int j = 0; j < kTile / kStep; ++j)
            copy16((at ^ copy_turn(j)) + j * 512, from_k + (PACKED ? j * 512 : (uint64_t)(j * kStep) * a.k_token_stride));
#pragma unroll
          for (int j = 0; j < kTile / kStep; ++j)
            copy16((at ^ copy_turn(j)) + kTile * D + j * 512, from_v + (PACKED ? j * 512 : (uint64_t)(j * kStep) * a.v_token_stride));
          if (lane < 2) copy4(scales + h * 8, scale + (uint64_t)p * (uint32_t)a.kv_heads);
          if (++sub == a.tiles_per_block) {
            sub = 0;
            ++block;
            page = next_page;
            next_page = page_at(a, s, block + 1);
          }
        }
        ++unit;
      }
      copy_commit();
    }
  };

  // A warp's running sums over the units of one segment.
  struct Rows {
    uint32_t q[kQShared ? 1 : NT][2 * kKWords];
    float o[NT][D / 16][4], m[NT][2], l[NT][2], factor[NT][2];
    // Tokens that every row sees are [most_low, least_high), those that some
    // row sees are within [least_low, most_high).
    int least_high, most_low, least_low, most_high;
    uint32_t unseen;  // rows (bits) of this lane's columns without a token yet, whose m is 0
    bool settled;     // no lane has any

    // `table` gets the segment's rows.
    __device__ __forceinline__ void begin(const AttendArgs& a, const Segment& s, uint32_t ring, int4* table) {
      const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
      int token, head, low = 0, high = 0;
      const bool there = lane < kRows && row_of(a, s, lane, token, head, low, high);
      if (lane < kRows) table[lane] = make_int4(there ? token : -1, head, low, high);
      __syncwarp();
      uint32_t mine[NT][2 * kKWords];
#pragma unroll
      for (int n = 0; n < NT; ++n) load_q(a, table[n * 8 + g], mine[n]);
      if (s.fresh == 1) {  // all rows are one query's
        least_high = most_high = s.length;
        least_low = most_low = a.window > 0 ? max(0, s.length - a.window) : 0;
      } else {
        least_high = __reduce_min_sync(0xffffffffu, there ? high : 0x7fffffff);
        least_low = __reduce_min_sync(0xffffffffu, there ? low : 0x7fffffff);
        most_low = __reduce_max_sync(0xffffffffu, low);
        most_high = __reduce_max_sync(0xffffffffu, high);
      }
      unseen = (1u << (2 * NT)) - 1u;
      settled = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) m[n][i] = l[n][i] = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float up = convert_q(a, mine[n]);
#pragma unroll
        for (int w = 0; w < kKWords; ++w) {
          if constexpr (kQShared) {  // each lane reads what it writes
            asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(ring + S * kStage + (n * kKWords + w) * 256 + lane * 8), "r"(mine[n][2 * w]), "r"(mine[n][2 * w + 1]) : "memory");
          } else {
            q[n][2 * w] = mine[n][2 * w];
            q[n][2 * w + 1] = mine[n][2 * w + 1];
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) factor[n][i] = a.scale_log2 * __shfl_sync(0xffffffffu, up, (2 * c + i) * 4);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][i][j] = 0.f;
    }

    // Rescales to the columns' new maxima; sc holds scores less m.
    __device__ __forceinline__ void grow(float (&sc)[MT][NT][4]) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = -INFINITY;
#pragma unroll
          for (int h = 0; h < MT; ++h) top = fmaxf(top, fmaxf(sc[h][n][i], sc[h][n][i + 2]));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          const uint32_t bit = 1u << (2 * n + i);
          float by = fmaxf(top - kTop, 0.f), f = exp2_approx(-by);
          if (unseen & bit) {  // its sums are zeros
            const bool some = top > -INFINITY;
            by = some ? top - kTop : 0.f;
            f = 0.f;
            if (some) unseen &= ~bit;
          }
          m[n][i] += by;
#pragma unroll
          for (int h = 0; h < MT; ++h) {
            sc[h][n][i] -= by;
            sc[h][n][i + 2] -= by;
          }
          l[n][i] *= f;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            o[n][d][i] *= f;
            o[n][d][i + 2] *= f;
          }
        }
      }
      settled = !__any_sync(0xffffffffu, unseen);
    }

    // The unit of tokens base.. of the segment in the stage at `at`; hidden: its
    // tiles (bits) whose pages are outside the pool.
    __device__ __forceinline__ void add(const int4* table, int base, uint32_t at, uint32_t ring, uint32_t hidden) {
      const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
      // Scores: [16 tokens][8 rows] for each tile of tokens and of rows, one tile
      // alone in two chains.
      constexpr int kChains = NT * MT == 1 ? 2 : 1;
      float sc[MT][NT][4], sd[4] = {0.f, 0.f, 0.f, 0.f}, v_inverse[MT];
      bool edge[MT], above = false;
#pragma unroll
      for (int h = 0; h < MT; ++h) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[h][n][i] = 0.f;
        const uint32_t at_k = at + h * kTileBytes + place(g, D == 64 ? c : 2 * c);
#pragma unroll
        for (int part = 0; part < kKWords / 4; ++part) {
          uint32_t k0[4], k1[4];
          const uint32_t from = (at_k ^ (part & 1) * 16) + (part >> 1) * 128;
          lds_words<4>(from, k0);
          lds_words<4>(from + 8 * D, k1);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t a0, a1, a2, a3;
            codes_to_half<E4M3>(k0[w], a0, a2);
            codes_to_half<E4M3>(k1[w], a1, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              uint32_t b[2];
              if constexpr (kQShared) {
                lds_words<2>(ring + S * kStage + (n * kKWords + 4 * part + w) * 256 + lane * 8, b);
              } else {
                b[0] = q[n][8 * part + 2 * w];
                b[1] = q[n][8 * part + 2 * w + 1];
              }
              mma16816(kChains == 2 && (w & 1) ? sd : sc[h][n], a0, a1, a2, a3, b[0], b[1]);
            }
          }
        }
      }
#pragma unroll
      for (int h = 0; h < MT; ++h) {
        const bool good = !(hidden >> h & 1);
        float k_scale, v_scale, v_log2;
        asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(k_scale), "=f"(v_scale) : "r"(at + kScales + h * 8));
        if (v_scale < kLeastScale) v_scale = kLeastScale;
        asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(v_log2) : "f"(v_scale));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(v_inverse[h]) : "f"(v_scale));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sc[h][n][i] = fmaf(kChains == 2 ? sc[h][n][i] + sd[i] : sc[h][n][i], factor[n][i & 1] * k_scale, v_log2 - m[n][i & 1]);
        }
        const int first = base + h * kTile;
        edge[h] = first + kTile > least_high || first < most_low || !good;  // the same in all lanes
        if (edge[h]) {
          // A unit of two tiles begins at a whole unit, so that its first may be a
          // page that the window hides wholly, scales of NaN and all.
          if (!good || (MT > 1 && (first + kTile <= least_low || first >= most_high))) v_inverse[h] = 0.f;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int2 sees = *reinterpret_cast<const int2*>(&table[n * 8 + 2 * c + i].z);
              const int low = sees.x, high = sees.y, t = first + g;
              if (t >= high || t < low || !good) sc[h][n][i] = -INFINITY;
              if (t + 8 >= high || t + 8 < low || !good) sc[h][n][i + 2] = -INFINITY;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
          above |= fmaxf(fmaxf(sc[h][n][0], sc[h][n][2]), fmaxf(sc[h][n][1], sc[h][n][3])) > kTop + kSlack;
      }
      if (__any_sync(0xffffffffu, above) || !settled) grow(sc);
      uint32_t pb[MT][NT][2];
#pragma unroll
      for (int h = 0; h < MT; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = exp2_approx(sc[h][n][i]);
          l[n][0] = fmaf(w[0] + w[2], v_inverse[h], l[n][0]);
          l[n][1] = fmaf(w[1] + w[3], v_inverse[h], l[n][1]);
          pb[h][n][0] = transpose8x8(pack_half2(w[0], w[1]));
          pb[h][n][1] = transpose8x8(pack_half2(w[2], w[3]));
        }
      constexpr int kPart = kVWords < 4 ? kVWords : 4;  // words of a load
#pragma unroll
      for (int h = 0; h < MT; ++h) {
        const uint32_t at_v = at + h * kTileBytes + kTile * D + (D == 64 ? place(2 * c, g >> 1) + (g & 1) * 8 : place(2 * c, D == 128 ? g : 2 * g));
#pragma unroll
        for (int part = 0; part < kVWords / kPart; ++part) {
          uint32_t v[4][kPart];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            lds_words<kPart>((at_v ^ ((j & 1) * kOdd) ^ (part * 16)) + (j & 1) * kOddRow + (j >> 1) * 8 * D, v[j]);
          if (edge[h]) {  // bytes of tokens that no row sees may be anything, e4m3's NaN too
            const int first = base + h * kTile, past = hidden >> h & 1 ? 0 : most_high - first, before = least_low - first;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int t = 2 * c + (j & 1) + (j >> 1) * 8;
              if (t >= past || t < before)
#pragma unroll
                for (int w = 0; w < kPart; ++w) v[j][w] = 0u;
            }
          }
#pragma unroll
          for (int w = 0; w < kPart; ++w) {
            uint32_t e[4], f[4];  // [channel 4w + i]: tokens (2c, 2c+1) and (2c+8, 2c+9)
            codes_to_half<E4M3>(prmt(v[0][w], v[1][w], 0x5140), e[0], e[1]);
            codes_to_half<E4M3>(prmt(v[0][w], v[1][w], 0x7362), e[2], e[3]);
            codes_to_half<E4M3>(prmt(v[2][w], v[3][w], 0x5140), f[0], f[1]);
            codes_to_half<E4M3>(prmt(v[2][w], v[3][w], 0x7362), f[2], f[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma16816(o[n][2 * (part * kPart + w)], e[0], e[1], f[0], f[1], pb[h][n][0], pb[h][n][1]);
              mma16816(o[n][2 * (part * kPart + w) + 1], e[2], e[3], f[2], f[3], pb[h][n][0], pb[h][n][1]);
            }
          }
        }
      }
    }

    __device__ __forceinline__ void finish() {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], d);
          if (unseen >> (2 * n + i) & 1) m[n][i] = kFarBelow;
        }
    }
  };

  // Channels of o[.][i][j] for lane row group g: 2i + (j >> 1) from g * (D / 8).
  __device__ static __forceinline__ void write_rows(const AttendArgs& a, const int4* table, const float (&o)[NT][D / 16][4],
                                                    const float (&m)[NT][2], const float (&l)[NT][2]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int2 at = *reinterpret_cast<const int2*>(&table[n * 8 + 2 * c + i]);
        if (at.x < 0) continue;
        const float f = l[n][i] > 0.f || l[n][i] != l[n][i] ? 1.f / l[n][i] : 0.f;
        const long long row = (long long)at.x * a.kv_heads * a.group + at.y;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
          store_row(a, row * D + g * (D / 8) + 4 * d,
                    make_float4(o[n][2 * d][i] * f, o[n][2 * d][i + 2] * f, o[n][2 * d + 1][i] * f, o[n][2 * d + 1][i + 2] * f));
        if (a.lse && g == 0) a.lse[row] = l[n][i] == 0.f ? -INFINITY : (m[n][i] + log2f(l[n][i])) * 0.69314718055994531f;
      }
  }

  // Where a joined row goes: its place among the rows of out (-1: the tile has
  // no such row), and what its sums are multiplied by.
  __device__ static __forceinline__ int row_place(const AttendArgs& a, const Segment& s, int row, float m, float l, float& by) {
    by = l > 0.f || l != l ? 1.f / l : 0.f;
    int token, head, low, high;
    if (!row_of(a, s, row, token, head, low, high)) return -1;
    const int at = token * a.kv_heads * a.group + head;
    if (a.lse) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
    return at;
  }
  __device__ static __forceinline__ void store_joined(const AttendArgs& a, int place, int d, const float4& x, float by) {
    if (place >= 0) store_row(a, (long long)place * D + d, make_float4(x.x * by, x.y * by, x.z * by, x.w * by));
  }

  static constexpr int kPartFloats = kRows * (D + 2);  // o, m, l of a CTA's part

  __device__ static __forceinline__ void add_part(const float4& y, float f, float4& x) {
    x.x = fmaf(y.x, f, x.x);
    x.y = fmaf(y.y, f, x.y);
    x.z = fmaf(y.z, f, x.z);
    x.w = fmaf(y.w, f, x.w);
  }

  __device__ static void run(const AttendArgs& a, Shared& sh, int* prefix) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_trigger();
    pdl_wait();
    int* lengths = prefix + a.requests + 1;
    int* starts = lengths + a.requests;
    const int most = (int)min((long long)a.max_blocks * a.block_size, 0x7fffffffLL);
    int carry = 0, longest = 0, segments = 0;
    for (int base = 0; base < a.requests; base += W * 32) {
      const int r = base + tid;
      int mine = 0, count = 0;
      if (r < a.requests) {
        const int length = min(max(ld_int(a.lengths + r), 0), most);
        int first = r, fresh = 1, unit0;
        if (a.starts) {
          first = ld_int(a.starts + r);
          const int next = ld_int(a.starts + r + 1);
          fresh = max(0, next - first);
          starts[r] = first;
          if (r == a.requests - 1) starts[r + 1] = next;
        }
        lengths[r] = length;
        const int tiles = tiles_of(a, first, fresh);
        if (tiles > 0) {
          const int one = units_of(a, length, fresh, unit0) + kStart;
          longest = max(longest, one);
          count = tiles * a.heads;
          mine = one * count;
        }
      }
      int sum = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += x;
      }
      longest = __reduce_max_sync(0xffffffffu, longest);
      count = __reduce_add_sync(0xffffffffu, count);
      if (lane == 31) {
        sh.total[warp] = sum;
        sh.longest[warp] = longest;
        sh.segments[warp] = count;
      }
      __syncthreads();
      int before = carry, all = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int x = sh.total[w];
        if (w < warp) before += x;
        all += x;
        longest = max(longest, sh.longest[w]);
        segments += sh.segments[w];
      }
      if (r < a.requests) prefix[r] = before + sum - mine;
      carry += all;
      if (tid == 0) prefix[a.requests] = carry;  // the last round's is the whole
      __syncthreads();
    }
    const int all = carry;
    if (all == 0) return;
    // Every CTA has the same number of places (the last has the rest), one for
    // each of its warps at least; CTA u / chunk has place u.  Nor is a segment
    // of n units cut in more than about sqrt(2 n) parts: one CTA joins them, at
    // a time for each that a warp needs for half a unit.  (Three requests of up
    // to 36 thousand tokens and one KV head: 30.7 -> 20.9 us.)  Where segments
    // are short the borders move to the nearest segment's, so that no segment
    // is shared between CTAs: joining one costs about as long as the units do
    // that a CTA gets too many.  (64 requests of up to 200 tokens 15.6 -> 12.0
    // us, of up to 1000 tokens 24.8 -> 21.6; from 2000 on it makes no odds.)  Few
    // segments would leave CTAs idle, though, and from 36 units on that costs more
    // than the joins: 8 KV heads of 128, us with moved borders / without, requests of
    //                 300 tokens  700        1000       1500
    //    1 (8 segments)  7.9/9.6   10.0/9.9  11.9/10.2  14.5/10.9
    //    8 (64)          9.5/11    13.2/12.4 15.9/13.2  20.4/15.1
    //   24 (192)         9.8/13    13.5/14.9 16.3/17.9  20.9/20.7
    //   64 (512)          13/17    21.0/24.4 28.6/32.7  39.1/42.2
    // so borders move there only if there are segments for half the CTAs.
    const int least = max(W, (int)sqrtf(0.5f * longest));
    const int grid = min((int)gridDim.x, (all + least - 1) / least);
    const int chunk = (all + grid - 1) / grid;
    const int cta = blockIdx.x;
    if (cta >= grid || cta * chunk >= all) return;
    const bool snap = longest <= kVeryShort || (longest <= kShort / MT && 2 * segments >= (int)gridDim.x);
    int cta0 = cta * chunk, cta1 = min(all, cta0 + chunk);
    if (snap) {
      if (warp < 2) {
        int x = warp ? cta1 : cta0;
        if (x > 0 && x < all) {
          const Segment s = segment_at(a, prefix, x);
          const int from = s.begin - kStart, to = s.begin + s.units;
          x = x - from <= to - x ? from : to;
        }
        if (lane == 0) sh.range[warp] = x;
      }
      __syncthreads();
      cta0 = sh.range[0];
      cta1 = sh.range[1];
      if (cta0 >= cta1) return;
    }
    const int u0 = cta0 + (cta1 - cta0) * warp / W, u1 = cta0 + (cta1 - cta0) * (warp + 1) / W;
    if (lane < 2) sh.used[2 * warp + lane] = 0;
    __syncwarp();

    if (u0 < u1) {
      const uint32_t ring = smem_u32(sh.ring[warp]);
      Segment& s = sh.now[warp];
      {
        const Segment t = segment_at(a, prefix, u0);
        if (lane == 0) s = sh.fed[warp] = t;
        __syncwarp();
      }
      Feed feed;
      feed.unit = u0;
      feed.end = u1;
      feed.to = ring + place(lane / kPieces, lane % kPieces);
      feed.hidden = 0;
      feed.enter(a, s);
#pragma unroll 1
      for (int i = 0; i < S - 1; ++i) feed.next(a, prefix, sh.fed[warp], i * kStage, i);
      Rows rows;
      int offset = 0, stage = 0, freed = (S - 1) * kStage, freed_stage = S - 1;
      for (int u = u0;;) {
        const int from = max(0, u - s.begin), to = min(s.units, u1 - s.begin);
        if (to <= 0) break;  // only the segment's start is this warp's
        rows.begin(a, s, ring, sh.rows[warp]);
        int base = (s.unit0 + from) * kUnit;
#pragma unroll 1
        for (int i = from; i < to; ++i) {
          copy_wait<S - 2>();
          __syncwarp();  // the unit is there for all lanes, and the stage before it has been read by all
          feed.next(a, prefix, sh.fed[warp], freed, freed_stage);
          rows.add(sh.rows[warp], base, ring + offset, ring, feed.hidden >> (stage * MT));
          base += kUnit;
          freed = offset;
          freed_stage = stage;
          offset += kStage;
          if (++stage == S) stage = offset = 0;
        }
        rows.finish();
        const int before = u;
        u = s.begin + to;
        if (from == 0 && to == s.units) {
          write_rows(a, sh.rows[warp], rows.o, rows.m, rows.l);
        } else {
          // An early part, after which the warp goes on, waits in L2; the last
          // one takes the place of the ring, where nothing is left to come.
          const bool early = u < u1;
          const int slot = 2 * warp + (early ? 0 : 1), g = lane >> 2, c = lane & 3;
          float* part = early ? a.early + (long long)(cta * W + warp) * kRows * D : reinterpret_cast<float*>(sh.ring[warp]);
          if (!early) __syncwarp();
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int row = n * 8 + 2 * c + i;
              float* p = part + row * D + g * (D / 8);
#pragma unroll
              for (int d = 0; d < D / 32; ++d)
                *reinterpret_cast<float4*>(p + 4 * d) =
                    make_float4(rows.o[n][2 * d][i], rows.o[n][2 * d][i + 2], rows.o[n][2 * d + 1][i], rows.o[n][2 * d + 1][i + 2]);
              if (g == 0) {
                sh.m[slot][row] = rows.m[n][i];
                sh.l[slot][row] = rows.l[n][i];
              }
            }
          if (lane == 0) {
            sh.seg[slot] = s;
            sh.used[slot] = 1;
          }
        }
        if (u >= u1 || u <= before) break;  // (the second: starts that do not rise)
        int r, which;
        after(a, prefix, s.request, s.which, u, r, which);
        __syncwarp();  // every lane has read s
        const Segment t = segment_of(a, prefix, r, which);
        if (lane == 0) s = t;
        __syncwarp();
      }
      copy_wait<0>();
    }
    __syncthreads();

    // Parts of one segment are neighbours among the used slots: a group.  This
    // code runs once a call, and fetching it costs more than running it: loops
    // are short and few.
    const int used = lane < kSlots ? sh.used[lane] : 0;
    const uint32_t valid = __ballot_sync(0xffffffffu, used);
    if (valid == 0) return;
    const int begin = used ? sh.seg[lane].begin : -1;
    const uint32_t below = valid & ((1u << lane) - 1u);
    const int prev = __shfl_sync(0xffffffffu, begin, below ? 31 - __clz(below) : 0);
    const uint32_t heads = __ballot_sync(0xffffffffu, used && (below == 0 || prev != begin));
    const int groups = __popc(heads), parts = __popc(valid);
    auto numbered = [&](int slot) { return __popc(valid & ((1u << slot) - 1u)); };  // among the used
    if (warp == 0 && used) {
      sh.part[__popc(below)] =
          lane & 1 ? reinterpret_cast<const float*>(sh.ring[lane >> 1]) : a.early + (long long)(cta * W + (lane >> 1)) * kRows * D;
      if (heads >> lane & 1) sh.group[__popc(heads & ((1u << lane) - 1u))] = __popc(below);
      if (lane == 31 - __clz(valid)) sh.group[groups] = parts;
    }
    // A group's rows, one a lane: their maxima, sums and parts' factors, and
    // where they go.
    uint32_t left = heads;
#pragma unroll 1
    for (int i = 0; i < groups; ++i, left &= left - 1) {
      if (i % W != warp) continue;
      const int first = __ffs(left) - 1;
      const uint32_t after = left & (left - 1);
      const uint32_t members = valid & ~((left & -left) - 1u) & (after ? (after & -after) - 1u : 0xffffffffu);
      // Lanes beyond the rows take other slots of the same rows.
      constexpr int P = 32 / kRows, N = (kSlots + P - 1) / P;
      const int row = lane % kRows, own = lane / kRows;
      float m[N], top = kFarBelow, l = 0.f;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int slot = k * P + own;
        m[k] = own < P && slot < kSlots && (members >> slot & 1) ? sh.m[slot][row] : -INFINITY;
        top = fmaxf(top, m[k]);
      }
#pragma unroll
      for (int d = kRows; P > 1 && d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int slot = k * P + own;
        if (m[k] > -INFINITY) {
          const float f = exp2_approx(m[k] - top);
          l = fmaf(f, sh.l[slot][row], l);
          sh.factor[numbered(slot)][row] = f;
        }
      }
#pragma unroll
      for (int d = kRows; P > 1 && d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
      if (lane >= kRows) continue;
      const Segment& s = sh.seg[first];
      if (s.begin >= cta0 && s.begin + s.units <= cta1) {
        sh.place[i][lane] = row_place(a, s, lane, top, l, sh.by[i][lane]);
      } else {  // a part of what several CTAs share
        const int which = cta * 2 + (s.begin >= cta0 ? 1 : 0);
        float* part = a.partials + (long long)which * kPartFloats;
        __stcg(part + kRows * D + lane, top);
        __stcg(part + kRows * D + kRows + lane, l);
        sh.place[i][lane] = -2 - which;
      }
    }
    __syncthreads();
    // A thread has U elements of four channels of each joined tile.
    constexpr int kQuads = kRows * D / 4, T = W * 32, U = kQuads > T ? kQuads / T : 1;
    static_assert(kQuads <= T || kQuads % T == 0, "");
    auto row_at = [&](int u) { return (tid + u * T) / (D / 4); };
    const int d = tid % (D / 4) * 4;
    static_assert(T % (D / 4) == 0, "a thread's elements lie in the same channels");
    const bool mine_too = tid < kQuads;
#pragma unroll 1
    for (int i = 0; i < groups; ++i) {
      if (!mine_too) break;
      const int end = sh.group[i + 1];
      float4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
      for (int k = sh.group[i]; k < end; ++k) {
        const float* from = sh.part[k] + d;
#pragma unroll
        for (int u = 0; u < U; ++u) add_part(*reinterpret_cast<const float4*>(from + row_at(u) * D), sh.factor[k][row_at(u)], x[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = row_at(u), place = sh.place[i][row];
        if (place >= -1) store_joined(a, place, d, x[u], sh.by[i][row]);
        else __stcg(reinterpret_cast<float4*>(a.partials + (long long)(-2 - place) * kPartFloats + row * D + d), x[u]);
      }
    }
    // The CTA's first and last segments may be shared with others: the last CTA
    // to arrive joins the parts in the order of the CTAs.
    if (snap) return;
    const int end_slot[2] = {__ffs(heads) - 1, 31 - __clz(heads)};
    const int ends = groups == 1 ? 1 : 2;
    __syncthreads();
    if (tid < 2) {
      const Segment& s = sh.seg[tid ? end_slot[1] : end_slot[0]];
      int last = 0;
      if (tid < ends && !(s.begin >= cta0 && s.begin + s.units <= cta1)) {
        const int c0 = s.begin / chunk, c1 = (s.begin + s.units - 1) / chunk;
        // With the barrier: the whole CTA's parts are seen before the count,
        // and the others' parts by the CTA that counts last.
        int before;
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(a.counters + c0) : "memory");
        if (before == c1 - c0) {
          last = c1 - c0 + 1;
          a.counters[c0] = 0;
        }
        sh.range[tid] = c0;
      }
      sh.last[tid] = last;
    }
    __syncthreads();
    const int n0 = sh.last[0], n1 = sh.last[1];  // parts to join, of the first and of the last segment
    if (n0 + n1 == 0) return;
    auto part = [&](int end, int i) { return a.partials + (long long)((sh.range[end] + i) * 2 + (i == 0 ? 1 : 0)) * kPartFloats; };
    // The parts' factors in place of the rings: a lane has a row, and the lanes
    // and warps beyond the rows other parts; then the rows' elements, of both
    // segments together.
    constexpr int P = 32 / kRows, G = W * P;
    float* sums = reinterpret_cast<float*>(sh.ring);  // [2][G][kRows]
    float* factor = sums + 2 * G * kRows;             // [n0 + n1][kRows]
    const int row = lane % kRows, mine = warp * P + lane / kRows;
    const bool busy = lane < P * kRows;
#pragma unroll 1
    for (int i = mine; i < n0 + n1; i += G) {
      const int end = i >= n0;
      if (busy) factor[i * kRows + row] = __ldcg(part(end, end ? i - n0 : i) + kRows * D + row);
    }
    __syncthreads();
    float top[2] = {kFarBelow, kFarBelow};
#pragma unroll 4
    for (int i = 0; i < n0 + n1; ++i) {
      const float m = factor[i * kRows + row];
      if (i < n0) top[0] = fmaxf(top[0], m); else top[1] = fmaxf(top[1], m);
    }
    __syncthreads();
    float l[2] = {0.f, 0.f};
#pragma unroll 1
    for (int i = mine; i < n0 + n1; i += G) {
      const int end = i >= n0;
      if (busy) {
        const float f = exp2_approx(factor[i * kRows + row] - (end ? top[1] : top[0]));
        const float add = f * __ldcg(part(end, end ? i - n0 : i) + kRows * D + kRows + row);
        if (end) l[1] += add; else l[0] += add;
        factor[i * kRows + row] = f;
      }
    }
    if (busy) {
      sums[mine * kRows + row] = l[0];
      sums[(G + mine) * kRows + row] = l[1];
    }
    __syncthreads();
    if (warp < 2 && lane < kRows) {
      float sum = 0.f;
#pragma unroll 4
      for (int i = 0; i < G; ++i) sum += sums[(warp * G + i) * kRows + lane];
      if (sh.last[warp]) sh.place[warp][lane] = row_place(a, sh.seg[warp ? end_slot[1] : end_slot[0]], lane, warp ? top[1] : top[0], sum, sh.by[warp][lane]);
    }
    __syncthreads();
    constexpr int kBatch = 16 / U;  // parts that a thread has on their way at once
#pragma unroll 1
    for (int end = 0; end < 2; ++end) {
      const int n = end ? n1 : n0;
      if (n == 0 || !mine_too) continue;
      const float* f = factor + (end ? n0 : 0) * kRows;
      float4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int i = 0; i < n; i += kBatch) {
        float4 y[kBatch][U];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (i + k < n) y[k][u] = __ldcg(reinterpret_cast<const float4*>(part(end, i + k) + row_at(u) * D + d));
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (i + k < n) add_part(y[k][u], f[(i + k) * kRows + row_at(u)], x[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) store_joined(a, sh.place[end][row_at(u)], d, x[u], sh.by[end][row_at(u)]);
    }
  }
};

template <int D, int NT, int MT, bool E4M3, bool PACKED, int W, int S, int MINB>
__global__ void __launch_bounds__(W * 32, MINB) k_attend(const __grid_constant__ AttendArgs a) {
  extern __shared__ __align__(128) unsigned char raw[];
  using A = Attend<D, NT, MT, E4M3, PACKED, W, S>;
  A::run(a, *reinterpret_cast<typename A::Shared*>(raw), reinterpret_cast<int*>(raw + sizeof(typename A::Shared)));
}

// Warps of a CTA, stages of a warp's ring, CTAs of an SM and tiles of a unit for
// each head size and number of row tiles, as the registers allow (q D/8 and o
// D/4 for each row tile) and as measured, each against its alternative:
//   128, one row tile: 16 warps with 2 stages 167 us for the longest case above,
//     with 3 stages 175, one CTA of 16 warps 167 (but 15.7 instead of 13.4 for
//     four requests of 3000 tokens), four CTAs of 4 172
//   64, one row tile: two tiles of tokens side by side 52 us for the window case,
//     one 58 to 61
//   more row tiles: one CTA of 8 warps (drafts 44 us, two of 4 47.6, when both
//     were slower)
constexpr int unit_tiles(int head_dim) { return head_dim == 64 ? 2 : 1; }
template <int D, int NT>
struct Shape;
template <> struct Shape<64, 1> { static constexpr int W = 8, S = 2, MINB = 2; };
template <> struct Shape<64, 2> { static constexpr int W = 12, S = 3, MINB = 1; };
template <> struct Shape<64, 4> { static constexpr int W = 8, S = 3, MINB = 1; };
template <> struct Shape<128, 1> { static constexpr int W = 8, S = 2, MINB = 2; };
template <> struct Shape<128, 2> { static constexpr int W = 8, S = 3, MINB = 1; };
template <> struct Shape<128, 3> { static constexpr int W = 8, S = 3, MINB = 1; };
template <> struct Shape<128, 4> { static constexpr int W = 8, S = 3, MINB = 1; };
template <> struct Shape<256, 1> { static constexpr int W = 8, S = 2, MINB = 1; };
template <> struct Shape<256, 2> { static constexpr int W = 8, S = 2, MINB = 1; };

// The workspace: a counter for each CTA that can run at once (in the same place
// for every shape: they stay zero between calls), two parts of its segments,
// and an early part for each of its warps.  Parts are written before they are read.
struct Workspace {
  size_t counters, partials, early;  // bytes
};
size_t counter_bytes(int sms) { return ((size_t)sms * 4 * sizeof(int) + 255) / 256 * 256; }
template <int D, int NT>
Workspace workspace_of(int sms) {
  using P = Shape<D, NT>;
  const size_t ctas = (size_t)sms * P::MINB, rows = 8 * NT;
  static_assert(P::MINB <= 4, "the counters' room");
  return {counter_bytes(sms), (ctas * 2 * rows * (D + 2) * sizeof(float) + 255) / 256 * 256,
          ctas * P::W * rows * D * sizeof(float)};
}

template <int D, int NT, bool E4M3, bool PACKED>
dk_status launch(const AttendArgs& call, cudaStream_t stream) {
  AttendArgs a = call;
  constexpr int W = Shape<D, NT>::W, MINB = Shape<D, NT>::MINB, S = Shape<D, NT>::S, MT = unit_tiles(D);
  using A = Attend<D, NT, MT, E4M3, PACKED, W, S>;
  const size_t per = (a.starts ? 3 : 2) * sizeof(int);  // of a request in shared memory
  const size_t smem = sizeof(typename A::Shared) + per * (size_t)(std::min(a.requests, kMaxRequests) + 1);
  static_assert(sizeof(typename A::Shared) + 3 * sizeof(int) * (kMaxRequests + 1) <= 227 * 1024,
                "a CTA fits the shared memory");
  auto kernel = k_attend<D, NT, MT, E4M3, PACKED, W, S, MINB>;
  const Workspace w = workspace_of<D, NT>(sm_count(-1));
  a.counters = static_cast<int*>(a.workspace);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + w.counters);
  a.early = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + w.counters + w.partials);
  static thread_local unsigned long long prepared = 0;  // devices whose limit is set
  const int device = current_device();
  if (device >= 64 || !(prepared >> device & 1)) {
    const size_t most = sizeof(typename A::Shared) + 3 * sizeof(int) * (kMaxRequests + 1);
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) {
      set_cuda_error(e, "cudaFuncSetAttribute");
      return DK_ERR_CUDA;
    }
    if (device < 64) prepared |= 1ull << device;
  }
  const int heads = call.heads;  // of a launch
  for (int r = 0; r < call.requests; r += kMaxRequests) {
    a.requests = std::min(kMaxRequests, call.requests - r);
    a.lengths = call.lengths + r;
    a.table = call.table + (long long)r * a.table_stride;
    long long row = 0;  // the launch's first in q
    if (call.starts) {
      a.starts = call.starts + r;
    } else {  // one query each: the rows move with the requests
      row = r;
      a.tokens = call.tokens - r;
    }
    for (int h = 0; h < a.kv_heads; h += heads) {
      a.heads = std::min(heads, a.kv_heads - h);
      const long long at = (row * a.kv_heads + h) * a.group;  // among the rows of out
      a.q = static_cast<const uint16_t*>(call.q) + row * a.q_token_stride + (long long)h * a.group * a.q_head_stride;
      a.out = static_cast<uint16_t*>(call.out) + at * D;
      a.lse = call.lse ? call.lse + at : nullptr;
      a.k = call.k + h * a.k_head_stride;
      a.v = call.v + h * a.v_head_stride;
      a.k_scale = call.k_scale + h;
      a.v_scale = call.v_scale + h;
      // No more CTAs than the table's width can keep busy.
      const long long most = (((long long)a.max_blocks * a.block_size + A::kUnit - 1) / A::kUnit + A::kStart) * a.heads *
                             (call.starts ? (long long)a.requests + (long long)call.tokens * a.group / A::kRows : (long long)a.requests * ((a.group + A::kRows - 1) / A::kRows));
      const int grid = (int)std::min<long long>(sm_count(device) * MINB, (most + W - 1) / W);
      const dk_status s = launch_early("dk_cache_attention", kernel, dim3(grid), dim3(W * 32), smem, stream, a);
      if (s != DK_OK) return s;
    }
  }
  return DK_OK;
}

// Tiles of eight rows that one pass over the cache serves: as many as a KV
// head's query rows fill, within what the registers hold.
int row_tiles(int head_dim, long long rows) {
  if (rows <= 8) return 1;
  if (rows <= 16 || head_dim == 256) return 2;
  return head_dim == 128 && (rows <= 24 || (rows > 32 && rows <= 48)) ? 3 : 4;
}

template <int D, int NT>
dk_status launch_code(const AttendArgs& a, bool e4m3, cudaStream_t stream) {
  const bool packed = a.k_token_stride == D && a.v_token_stride == D;
  if (e4m3) return packed ? launch<D, NT, true, true>(a, stream) : launch<D, NT, true, false>(a, stream);
  return packed ? launch<D, NT, false, true>(a, stream) : launch<D, NT, false, false>(a, stream);
}

}  // namespace
}  // namespace dk

using namespace dk;

extern "C" size_t dk_cache_attention_workspace_bytes(int head_dim) {
  const int sms = sm_count(-1);
  auto all = [](const Workspace& w) { return w.counters + w.partials + w.early; };
  if (head_dim == 64) return std::max(all(workspace_of<64, 2>(sms)), all(workspace_of<64, 4>(sms)));
  if (head_dim == 128) return std::max(all(workspace_of<128, 2>(sms)), all(workspace_of<128, 4>(sms)));
  if (head_dim == 256) return all(workspace_of<256, 2>(sms));
  return 0;
}

extern "C" size_t dk_cache_attention_counter_bytes(void) { return counter_bytes(sm_count(-1)); }

extern "C" dk_status dk_cache_attention(const dk_cache_attention_args* p, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  if (!p) return DK_ERR_INVALID_ARG;
  const dk_cache8& c = p->cache;
  if (c.block_size < 16 || c.block_size > 256 || c.block_size % 16 || c.blocks < 1 || c.kv_heads < 1 ||
      p->q_heads < 1 || p->q_heads % c.kv_heads || p->requests < 0 || p->tokens < 0 || p->max_blocks < 1 ||
      p->window < 0 || (p->window > 0 && !p->causal))
    return DK_ERR_INVALID_ARG;
  if (c.code != DK_INT8 && c.code != DK_E4M3) return DK_ERR_INVALID_ARG;
  if (p->dtype != DK_FP16 && p->dtype != DK_BF16) return DK_ERR_INVALID_ARG;
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return DK_ERR_UNSUPPORTED;
  if (!p->starts && p->tokens != p->requests) return DK_ERR_INVALID_ARG;
  if (p->requests == 0 || p->tokens == 0) return DK_OK;
  if (!p->q || !p->out || !p->block_table || !p->lengths || !c.k || !c.v || !c.k_scale || !c.v_scale)
    return DK_ERR_INVALID_ARG;
  auto aligned = [](const void* x, uintptr_t n) { return reinterpret_cast<uintptr_t>(x) % n == 0; };
  const long long strides[] = {c.k_block_stride, c.k_head_stride, c.k_token_stride,
                               c.v_block_stride, c.v_head_stride, c.v_token_stride};
  for (long long s : strides)
    if (s < 0 || s % 32) return DK_ERR_INVALID_ARG;
  if (!aligned(c.k, 32) || !aligned(c.v, 32) || !aligned(p->q, 16) || !aligned(p->out, 16) ||
      p->q_token_stride % 8 || p->q_head_stride % 8)
    return DK_ERR_INVALID_ARG;
  // A page's stride and the offsets within one are kept in 32 bits.
  if (c.k_block_stride > INT32_MAX || c.v_block_stride > INT32_MAX ||
      c.k_token_stride > INT32_MAX / c.block_size || c.v_token_stride > INT32_MAX / c.block_size)
    return DK_ERR_UNSUPPORTED;
  // The line of units is counted in 32 bits, whatever the lengths turn out to be:
  // a launch takes as many KV heads as fit it.
  const int group = p->q_heads / c.kv_heads;
  const int nt = row_tiles(c.head_dim, ((long long)p->tokens + p->requests - 1) / p->requests * group);
  const int unit = kTile * unit_tiles(c.head_dim);
  const long long width = (long long)p->max_blocks * c.block_size, units = (width + unit - 1) / unit + 2;  // and a start's places
  const long long tiles = (long long)std::min(p->requests, kMaxRequests) + (long long)p->tokens * group / (8 * nt);
  if (width > INT32_MAX - 64 || (long long)p->tokens * p->q_heads > INT32_MAX || tiles > INT32_MAX / 2 / units) return DK_ERR_UNSUPPORTED;
  const size_t need = dk_cache_attention_workspace_bytes(c.head_dim);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 256)) return DK_ERR_WORKSPACE;

  AttendArgs a;
  a.q = p->q;
  a.k = static_cast<const uint8_t*>(c.k);
  a.v = static_cast<const uint8_t*>(c.v);
  a.k_scale = c.k_scale;
  a.v_scale = c.v_scale;
  a.table = p->block_table;
  a.lengths = p->lengths;
  a.starts = p->starts;
  a.out = p->out;
  a.lse = p->lse;
  a.workspace = workspace;
  a.q_token_stride = p->q_token_stride;
  a.q_head_stride = p->q_head_stride;
  a.k_block_stride = (uint32_t)c.k_block_stride;
  a.k_head_stride = c.k_head_stride;
  a.k_token_stride = (uint32_t)c.k_token_stride;
  a.v_block_stride = (uint32_t)c.v_block_stride;
  a.v_head_stride = c.v_head_stride;
  a.v_token_stride = (uint32_t)c.v_token_stride;
  a.table_stride = p->table_stride;
  a.max_blocks = p->max_blocks;
  a.blocks = c.blocks;
  a.block_size = c.block_size;
  a.tiles_per_block = c.block_size / kTile;
  a.requests = p->requests;
  a.tokens = p->tokens;
  a.kv_heads = c.kv_heads;
  a.heads = (int)std::min<long long>(c.kv_heads, INT32_MAX / 2 / units / tiles);
  a.group = group;
  auto magic = [](int by) { return by > 1 ? (unsigned)(((1ull << 32) + by - 1) / by) : 0u; };
  a.group_magic = magic(group);
  a.block_magic = magic(a.tiles_per_block);
  a.scale_log2 = p->scale * 1.4426950408889634f;
  a.causal = p->causal;
  a.window = p->window;
  a.bf16 = p->dtype == DK_BF16;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool e4m3 = c.code == DK_E4M3;
  switch (c.head_dim * 8 + nt) {
    case 64 * 8 + 1: return launch_code<64, 1>(a, e4m3, st);
    case 64 * 8 + 2: return launch_code<64, 2>(a, e4m3, st);
    case 64 * 8 + 4: return launch_code<64, 4>(a, e4m3, st);
    case 128 * 8 + 1: return launch_code<128, 1>(a, e4m3, st);
    case 128 * 8 + 2: return launch_code<128, 2>(a, e4m3, st);
    case 128 * 8 + 3: return launch_code<128, 3>(a, e4m3, st);
    case 128 * 8 + 4: return launch_code<128, 4>(a, e4m3, st);
    case 256 * 8 + 1: return launch_code<256, 1>(a, e4m3, st);
    default: return launch_code<256, 2>(a, e4m3, st);
  }
}
