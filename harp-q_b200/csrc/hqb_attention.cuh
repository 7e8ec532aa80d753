// Work division of the tree attention, shared by its kernels.
//
// An item is (request, key head, row tile): the row tile's query rows (row = node * group + head
// in group, so every row of the tile reads the same keys) against the request's keys, which are
// cut into blocks (64 or 128 keys): first the cached context, then the drafted nodes (the last block of
// either may be partly filled).  Items lie in order request, key head, row tile; the blocks of
// all items in that order are dealt to the CTAs in equal contiguous ranges, so ragged lengths
// balance whatever their order.  An item that spans CTAs leaves one partial result per CTA
// (unnormalised FP32 sums, running maximum and sum of weights) in the workspace, which
// attention_join_kernel joins in CTA order: the result depends on the grid, never on timing.
#pragma once

#include "hqb_serve.cuh"

namespace hqb {

// Quotients by a number that the host knows (Granlund and Montgomery, 1994), for n < 2^31: with
// s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1, n / d = (n + floor(m n / 2^32)) >> s.  Four
// instructions; the kernels' single warps that place copies waited for the usual thirty.
struct Divisor {
  uint32_t m, s;
  static Divisor of(uint32_t d) {
    Divisor v{0, 0};
    while (v.s < 31 && (1u << v.s) < d) ++v.s;
    v.m = static_cast<uint32_t>((((1ull << v.s) - d) << 32) / d) + 1;
    return v;
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (n + __umulhi(m, n)) >> s; }
};

struct Split;

// The softmax's reference for the exponent lies kWeightShift below the maximum, so that the weights reach
// up to 2^15.9 in FP16.  They are rounded to the type for the product with the values, and FP16 ends at
// 2^-24: weights up to 1 would lose what is below 2^-25 of the largest, from the product alone, and keys of
// that size that are many would be missing from the result.  So they keep all their bits down to 2^-27
// of the largest, and end at 2^-38.  BF16 has FP32's range.
template <typename T>
constexpr bool kNarrow = Elem<T>::kExpMask == 0x7C00u;
// log2 of how far the tensor-memory kernel lets the maximum outgrow its reference before it rescales sums.
// FP16: what the type has room for (2^15.9 < 65504).  32 trees of up to 64 nodes over up to 8192 tokens, FP16,
// by 2 338 us, by 2.9 324 us (by 8 with weights up to 2^8, which lose small ones, 322 us).
template <typename T>
constexpr float kSlack = kNarrow<T> ? 2.9f : 8.0f;
template <typename T>
constexpr float kWeightShift = kNarrow<T> ? 13.0f : 0.0f;

struct AttnParams {
  hqb_attention_args a;
  hqb_paged_cache c;
  int* error;
  Split* splits;       // [cta] the item that begins in the CTA and ends in a later one
  float* parts;         // [cta][2] partial results: see part_sums
  uint32_t group;       // query heads per key head
  uint32_t rows;        // rows of a row tile
  uint32_t block_shift; // log2 of the keys of a block
  Divisor by_page, by_group, by_rows;
  uint32_t dim_pad;     // padded head dimension (columns of a partial row)
  uint32_t min_blocks;  // fewest blocks worth a CTA of its own
  uint32_t whole;       // 1: items are not cut (a unit is an item, no partials)
  uint32_t grid;        // CTAs of the attention kernel
  uint32_t warps;       // of a CTA of the rows kernel
  uint32_t vec;         // 16-byte accesses fit every row
  float scale_log2;     // scale * log2(e)
};

// What attention_join_kernel has to know of an item whose parts are in CTAs c .. last.
struct Split {
  uint32_t last;  // c itself: nothing to join
  uint32_t start, nodes, head, tile;
  uint32_t pad[3];
};

struct Request {
  uint32_t start, nodes, ctx;
  uint32_t cached_blocks, blocks;  // blocks: 0 for a request without nodes
  uint32_t tiles;
};

__device__ __forceinline__ Request load_request(const AttnParams& p, uint32_t r, uint32_t& bad) {
  Request q;
  const int32_t s0 = p.a.starts[r], s1 = p.a.starts[r + 1];
  const int32_t c = p.a.context_lens[r];
  const uint32_t cap = p.a.tokens;
  q.start = s0 < 0 ? 0u : min(static_cast<uint32_t>(s0), cap);
  const uint32_t end = s1 < 0 ? 0u : min(static_cast<uint32_t>(s1), cap);
  q.nodes = end > q.start ? end - q.start : 0u;
  if (s0 < 0 || s1 < s0 || static_cast<uint32_t>(s1) > cap || q.nodes > p.a.max_new || c < 0) bad |= HQB_DEVERR_INDEX;
  q.nodes = min(q.nodes, p.a.max_new);
  q.ctx = static_cast<uint32_t>(max(c, 0));
  const uint64_t room = static_cast<uint64_t>(p.a.table_stride) * p.c.page_size;
  if (q.ctx > room) {
    bad |= HQB_DEVERR_PAGES;
    q.ctx = static_cast<uint32_t>(room);
  }
  const uint32_t over = (1u << p.block_shift) - 1;
  q.cached_blocks = (q.ctx + over) >> p.block_shift;
  q.blocks = q.nodes == 0 ? 0u : q.cached_blocks + ((q.nodes + over) >> p.block_shift);
  q.tiles = p.by_rows.quotient(q.nodes * p.group + p.rows - 1);
  return q;
}

__device__ __forceinline__ uint64_t request_units(const AttnParams& p, const Request& q) {
  return static_cast<uint64_t>(q.tiles) * p.c.kv_heads * (p.whole ? 1u : q.blocks);
}

// 64-bit quotients cost a few hundred cycles; nearly all of them fit 32 bits.
__device__ __forceinline__ uint64_t quotient(uint64_t a, uint64_t b) {
  return (a | b) >> 32 == 0 ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}

// CTAs that get units: at least min_blocks each, so that short work is not cut into pieces
// smaller than the cost of joining them.
__device__ __forceinline__ uint32_t busy_ctas(const AttnParams& p, uint64_t units) {
  const uint64_t most = p.whole ? units : quotient(units + p.min_blocks - 1, p.min_blocks);
  return static_cast<uint32_t>(most < p.grid ? most : p.grid);
}

__device__ __forceinline__ uint64_t first_unit(uint32_t cta, uint64_t units, uint32_t ctas) {
  return quotient(units * cta, ctas);
}
// The CTA whose range [first_unit(i), first_unit(i + 1)) holds unit u.
__device__ __forceinline__ uint32_t cta_of_unit(uint64_t u, uint64_t units, uint32_t ctas) {
  return static_cast<uint32_t>(quotient((u + 1) * ctas - 1, units));
}

// A CTA's walk over its units, one segment (a range of one item's blocks) at a time.  Every
// thread keeps its own copy; begin() is called by whole warps.
struct Walk {
  uint64_t left;         // units not yet handed out
  uint64_t units, past;  // of the whole call; the first after this CTA's
  uint32_t ctas;
  uint32_t r, head, tile, unit;
  Request q;
  // the current segment
  uint32_t b0, b1;

  __device__ __forceinline__ bool begin(const AttnParams& p, uint32_t cta, uint32_t& bad) {
    const uint32_t lane = threadIdx.x & 31;
    uint64_t mine = 0, inc = 0;  // inc: inclusive sum of a round of 32 requests
    units = 0;
    auto round = [&](uint32_t r0) {
      mine = r0 + lane < p.a.requests ? request_units(p, load_request(p, r0 + lane, bad)) : 0;
      inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= static_cast<uint32_t>(o)) inc += up;
      }
    };
    for (uint32_t r0 = 0; r0 < p.a.requests; r0 += 32) {
      round(r0);
      units += __shfl_sync(0xffffffffu, inc, 31);
    }
    ctas = busy_ctas(p, units);
    left = 0;
    if (cta >= ctas) return false;
    const uint64_t u0 = first_unit(cta, units, ctas);
    past = first_unit(cta + 1, units, ctas);
    left = past - u0;
    // the request that holds unit u0
    uint64_t carry = 0;
    for (uint32_t r0 = 0; r0 < p.a.requests; r0 += 32) {
      if (p.a.requests > 32) round(r0);  // else the one round's sums are at hand
      const uint32_t past = ballot(carry + inc > u0);
      if (past != 0) {
        const uint32_t at = __ffs(past) - 1;
        const uint64_t skip = u0 - (carry + __shfl_sync(0xffffffffu, inc - mine, at));
        r = r0 + at;
        q = load_request(p, r, bad);
        const uint32_t per_item = p.whole ? 1u : q.blocks;
        const uint64_t item = quotient(skip, per_item);
        unit = static_cast<uint32_t>(skip - item * per_item);
        head = static_cast<uint32_t>(quotient(item, q.tiles));
        tile = static_cast<uint32_t>(item - static_cast<uint64_t>(head) * q.tiles);
        return true;
      }
      carry += __shfl_sync(0xffffffffu, inc, 31);
    }
    return false;
  }

  // Sets b0, b1 to the next segment's blocks; r, head, tile and q name its item.
  __device__ __forceinline__ void open(const AttnParams& p) {
    if (p.whole) {
      b0 = 0;
      b1 = q.blocks;
      left -= 1;
    } else {
      b0 = unit;
      const uint64_t n = q.blocks - unit;
      b1 = unit + static_cast<uint32_t>(n < left ? n : left);
      left -= b1 - b0;
    }
  }
  // After a segment: the next item, unless the range ended inside this one.
  __device__ __forceinline__ void advance(const AttnParams& p, uint32_t& bad) {
    unit = 0;
    if (left == 0) return;
    if (++tile < q.tiles) return;
    tile = 0;
    if (++head < p.c.kv_heads) return;
    head = 0;
    do {  // a later request has the units that are left
      ++r;
      q = load_request(p, r, bad);
    } while (q.tiles == 0 && r + 1 < p.a.requests);
  }
  __device__ __forceinline__ bool complete() const { return b0 == 0 && b1 == q.blocks; }
};

// Writes down a CTA's split item: every CTA once, by one thread, after begin().  Only a CTA's last
// item can begin in it and end in a later one.
__device__ __forceinline__ void note_split(const AttnParams& p, Walk w, uint32_t cta, bool work, uint32_t& bad) {
  Split s{};
  s.last = cta;
  if (work) {
    const uint32_t begun = w.unit;  // blocks of the first item that lie in earlier CTAs
    bool head_of_item = begun == 0;
    uint64_t left = w.left;
    while (left > w.q.blocks - w.unit) {
      left -= w.q.blocks - w.unit;
      w.left = left;
      w.advance(p, bad);
      head_of_item = true;
    }
    uint64_t rest = w.q.blocks - w.unit - left;  // the item's blocks in later CTAs
    if (head_of_item && rest != 0) {
      s.start = w.q.start, s.nodes = w.q.nodes, s.head = w.head, s.tile = w.tile;
      s.last = cta_of_unit(w.past + rest - 1, w.units, w.ctas);
    }
  }
  p.splits[cta] = s;
}

// A partial result: sums [dim_pad / 4][rows][4] (neighbouring rows' 16 bytes adjacent, as a thread a
// row stores them) and statistics [rows] {maximum, sum of weights}.  Of a CTA's two, slot 1 is that
// of an item that begins in it, 0 that of one that began before.
__device__ __forceinline__ float* part_sums(const AttnParams& p, uint32_t cta, uint32_t slot) {
  return p.parts + (static_cast<uint64_t>(cta) * 2 + slot) * p.rows * (p.dim_pad + 2);
}
__device__ __forceinline__ float2* part_stats(const AttnParams& p, uint32_t cta, uint32_t slot) {
  return reinterpret_cast<float2*>(part_sums(p, cta, slot) + p.rows * p.dim_pad);
}

// Address of one cached key's row in k or v (elements from the base), its page checked.
__device__ __forceinline__ uint64_t key_offset(const AttnParams& p, const int32_t* table, uint32_t key, uint32_t head,
                                               uint32_t& bad) {
  const uint32_t column = p.by_page.quotient(key), inside = key - column * p.c.page_size;
  uint32_t page = static_cast<uint32_t>(table[column]);
  if (page >= p.c.num_pages) {
    bad |= HQB_DEVERR_PAGES;
    page = 0;
  }
  return page * p.c.page_stride + inside * p.c.token_stride + head * p.c.head_stride;
}

// 32 bits of the nodes that node `node` of request q sees among nodes 32*word ..
__device__ __forceinline__ uint32_t node_mask(const AttnParams& p, const Request& q, uint32_t node, uint32_t word) {
  uint32_t bits;
  if (p.a.mask != nullptr) {
    bits = p.a.mask[static_cast<uint64_t>(q.start + node) * p.a.mask_words + word];
  } else {
    const int32_t n = static_cast<int32_t>(node) + 1 - static_cast<int32_t>(word * 32);  // nodes 0 .. node
    bits = n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u;
  }
  const int32_t live = static_cast<int32_t>(q.nodes) - static_cast<int32_t>(word * 32);
  return live >= 32 ? bits : live <= 0 ? 0u : bits & ((1u << live) - 1u);
}

// Launches attention_tmem_kernel (hqb_attention_tmem.cu): p.rows 2 * (128 / group * group), p.block_shift 7, p.dim_pad 64 or 128.
template <typename T>
cudaError_t launch_attention_tmem(const AttnParams& p, cudaStream_t st);

}  // namespace hqb
