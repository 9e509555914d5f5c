// chunk.cu -- attention of a chunk of new tokens over the paged key-value
// cache: pieces of prompts, whole prompts, drafted tokens, single tokens.
//
// out_i = softmax(scale q_i K^T) V over the slots row i sees, one pass over K
// and V with the running maximum and sum of each row.  4 D FLOP a (query, head,
// slot) against 4 D bytes a (kv head, slot) in 16 bits: the tensor cores bound
// it from some 250 packed query rows a kv head on, HBM below that.
//
// 16-bit types.  The query heads of a kv head share its K and V, so their rows
// are packed: a tile of 128 rows holds 128 / G tokens x G heads.  A unit
// (sequence, kv head, up to two tiles of tokens) streams the slots that its last
// token sees in blocks of 128.  All units' blocks, in order, are dealt out as
// equal runs, whatever the lengths, to one CTA per SM; a unit that spans CTAs
// leaves unnormalised parts in the workspace, which a second kernel joins in
// the order of the run.  Inside a CTA the roles are those of the prompt's own
// attention (attn_fwd.cu): a warp each issues the TMA loads of Q and K and of V, one the
// tcgen05 products, two warpgroups hold a query row a thread and do the softmax.  A unit of two tiles
// gives each warpgroup one of them; a unit of one gives them its blocks in
// turn, and their two results meet in shared memory at its end.
// TMEM (512 columns): S0 [0,128) S1 [128,256) O0 [256,256+D) O1 [256+D,256+2D),
// P as 16-bit pairs over the first half of S.
//
// Measured: 2 x 1.5-1.8 k tokens over 14-16 k, 64/8 heads of 128, bf16: 1755-1800 us
// (SM clock 1.66-1.6 GHz under the power limit), 890-865 TFLOP/s (2.6 us a block of
// 256 rows x 128 slots; the chain S, softmax, P V bounds it, as it does the prompt's
// own attention).  8 x 3-6 tokens over 12-16 k (471 MB): 101-107 us, 0.67-0.71 of
// HBM.  32 ragged sequences up to 2048 with 1-100 tokens, 32/8 x 64: 92 us: 8 us
// until the first scores, 4-5 a unit.  fp32, 3 x 1-129 tokens over 300-1025, 16 heads of 128: 154 us, with issue
// slots 42 % and the FMA pipe 27 % busy: eight warps an SM do not fill them.  A warp
// a (row, head), slot by slot, took 309 ms, 92 ms, 9.0 ms and 0.9 ms.
#include "tkb_common.cuh"
#include "../../include/tkm_b200.h"

namespace tkb {

// Lets the next launch of the stream come up from here on, when all CTAs of this
// one have started; its grid_wait() still waits for this one's end.
TKB_DEVFN void grid_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// What the deal reckons with: a block of a unit of two tiles, of one, of one of
// at most 16 rows; a unit on top (its queries' load, its rows' output); and a
// CTA's run at least, unless it has a unit of its own (shorter parts cost more
// to join than they save).  In 16 bits a block of one tile is a warpgroup's, of
// two both's; in fp32 the rows' products are what takes time.  Other 16-bit weights,
// us for 32 ragged sequences, 8 x 3-6 tokens over 12-16 k, 8 prompts of 1000-2048:
//   as below 92, 100, 186      unit 0   135, 103, 214    unit 2  99, 102, 195
//   unit 8   92,  98, 187      pair 1    96, 102, 190    one 2   99, 136, 190
// least: one sequence of 5 tokens over 333 16 us, 20 with 4, 16 with 24; the others
// are the same with 4 to 48.
struct ChunkCost {
  int pair, one, few, unit, least;
};
constexpr ChunkCost kCost16 = {2, 1, 1, 4, 12}, kCost32 = {8, 4, 1, 2, 8};

struct alignas(64) ChunkParams {
  CUtensorMap tmQ, tmK, tmV;  // 16-bit types
  tkb_kv_cache c;
  const void* q;
  void* out;
  float* lse;
  const int32_t* row_start;
  long long q_stride, out_stride;
  int rows, Hq, G;
  int gb, hb;          // query heads per tile, blocks of them per kv head (G <= hb * gb)
  int tt;              // tokens per tile: 128 / gb, of fp32 64 / gb
  int gran;            // slots per TMA box: what divides both a page and a block of 128
  ChunkCost cost;
  float scale_log2;
  float4* part;        // [2 * grid][2 tiles][D / 4][128 rows] unnormalised parts
  float2* part_ml;     // [2 * grid][2][128] their maxima (in powers of 2) and sums
  int4* span;          // [grid] what the CTA left: ChunkSpan bits, sequence, head group, unit
};

// The rows of sequence b: first row and number, inside [0, rows).
TKB_DEVFN void chunk_rows(const int32_t* row_start, int rows, int b, int& first, int& n) {
  if (!row_start) {
    first = b;
    n = 1;
    return;
  }
  int lo = row_start[b], hi = row_start[b + 1];
  if (lo < 0 || hi < lo || hi > rows) {
    atomicOr(&g_device_error, ERR_BAD_INDEX);
    lo = min(max(lo, 0), rows);
    hi = min(max(hi, lo), rows);
  }
  first = lo;
  n = hi - lo;
}

// ============================================================ the deal
constexpr int kChunkGrid = 148;   // one CTA per SM
constexpr int kChunkBlock = 128;  // slots per block

// A sequence: its rows, how many slots its first row sees less one (may be
// negative), what it holds, and its units.
struct ChunkSeq {
  int first, n, base, held;
  int units;
};
TKB_DEVFN int chunk_blocks(int base, int upto) {  // blocks for a row that sees base + upto slots; at least one
  return 1 + (max(base, 0) + upto - 1) / kChunkBlock;
}
// Cost of the first u (full) units: the sum over v < u of floor((per v + c) / 128), from the sum of the dividends and that
// of their remainders, which repeat after 128 / gcd(per, 128) terms, taking each value of their class mod the gcd once.
__noinline__ __device__ long long chunk_cost_before(const ChunkParams& p, int base, int u) {
  const int per = 2 * p.tt;
  const int c = max(base, 0) + per - 1, g = min(per & -per, kChunkBlock), period = kChunkBlock / g;
  const int turns = u / period;
  int rest = 0;
  long long rests = static_cast<long long>(turns) * (period * (c & (g - 1)) + g * (period * (period - 1) / 2));
#pragma unroll 1
  for (int v = turns * period; v < u; ++v) rest += (per * v + c) & (kChunkBlock - 1);
  rests += rest;
  const long long n = u, sum = (per * (n * (n - 1) / 2) + n * c - rests) / kChunkBlock;
  return n * (p.cost.unit + p.cost.pair) + p.cost.pair * sum;
}
TKB_DEVFN int chunk_block_cost(const ChunkParams& p, int tokens) {
  return tokens > p.tt ? p.cost.pair : tokens * p.gb > 16 ? p.cost.one : p.cost.few;
}
TKB_DEVFN int chunk_cost(const ChunkParams& p, const ChunkSeq& s, int u) {
  const int t0 = u * 2 * p.tt, tokens = min(2 * p.tt, s.n - t0);
  return p.cost.unit + chunk_block_cost(p, tokens) * chunk_blocks(s.base, t0 + tokens);
}
TKB_DEVFN ChunkSeq chunk_seq(const ChunkParams& p, int b) {
  ChunkSeq s;
  const int held = max(p.c.seq_lens[b], -(1 << 30)), most = p.c.max_pages * p.c.page_size;
  chunk_rows(p.row_start, p.rows, b, s.first, s.n);
  // rows without a slot see none, rows past the table all of it
  if (held < s.n || held > most) {
    if (s.n) atomicOr(&g_device_error, ERR_BAD_INDEX);
  }
  s.held = min(max(held, 0), most);
  s.base = min(held, most + s.n) - s.n;
  s.units = (s.n + 2 * p.tt - 1) / (2 * p.tt);
  return s;
}
TKB_DEVFN long long chunk_seq_cost(const ChunkParams& p, const ChunkSeq& s) {  // of one head group
  return s.n ? chunk_cost_before(p, s.base, s.units - 1) + chunk_cost(p, s, s.units - 1) : 0;
}

// One unit's share of a CTA's run.
struct ChunkItem {
  ChunkSeq s;
  int more;                // 0: the run has ended
  int b, hg, u;            // sequence, head group (kv head, block of query heads), unit of the sequence
  int t0, tokens;          // its tokens among the sequence's rows
  int nb0, nb1;            // blocks of its tiles (the second's are all the unit's)
  int jb, je;              // the run's blocks
  TKB_DEVFN bool pair(const ChunkParams& p) const { return tokens > p.tt; }  // two tiles
  TKB_DEVFN bool whole() const { return jb == 0 && je == nb1; }
};
// Walks the items of a run.  Every warp walks for itself, its state in shared
// memory: a lane steps it, ahead of its use, and the registers are the softmax's.
struct ChunkWalk {
  ChunkItem it[2];
  int b, hg, u, k;
  long long at, x0, x1;    // cost where the unit starts, where the run does and ends
  int count[6];            // what the warp has counted when its run is done, for a second walk
  // The item at hand; of the one after it once ahead() has been called.
  TKB_DEVFN const ChunkItem& item() const { return it[k & 1]; }
  TKB_DEVFN void step(const ChunkParams& p) {  // one lane: the item after the one at hand
    const int from = k & 1;
    ChunkSeq s = it[from].s;
    int b_ = b, hg_ = hg, u_ = u;
    long long at_ = at;
    const long long x0_ = x0, x1_ = x1;
    ChunkItem n;
    n.more = 0;
    while (at_ < x1_) {
      if (u_ == s.units) {
        u_ = 0;
        if (++hg_ == p.c.Hkv * p.hb) {
          hg_ = 0;
          do {
            if (++b_ >= p.c.B) break;
            s = chunk_seq(p, b_);
          } while (s.n == 0);
          if (b_ >= p.c.B) break;
        }
      }
      n.u = u_;
      n.t0 = u_ * 2 * p.tt;
      n.tokens = min(2 * p.tt, s.n - n.t0);
      const int each = chunk_block_cost(p, n.tokens);
      n.nb0 = chunk_blocks(s.base, n.t0 + min(n.tokens, p.tt));
      n.nb1 = chunk_blocks(s.base, n.t0 + n.tokens);
      const int cost = p.cost.unit + each * n.nb1;
      auto block_at = [&](long long x) {  // first block that starts at cost x of the unit or later
        if (x <= p.cost.unit) return 0;
        if (x >= cost) return n.nb1;
        return (static_cast<int>(x) - p.cost.unit + each - 1) / each;
      };
      n.jb = block_at(x0_ - at_);
      n.je = block_at(x1_ - at_);
      at_ += cost;
      ++u_;
      if (n.jb < n.je) {
        n.more = 1;
        break;
      }
    }
    n.s = s;
    n.b = b_;
    n.hg = hg_;
    it[from ^ 1] = n;
    b = b_;
    hg = hg_;
    u = u_;
    at = at_;
  }
  TKB_DEVFN void ahead(const ChunkParams& p) {  // a whole warp
    if (lane_id() == 0) step(p);
  }
  TKB_DEVFN bool next() {  // a whole warp, after ahead()
    __syncwarp();
    const int now = k + 1;
    __syncwarp();
    if (lane_id() == 0) k = now;
    __syncwarp();
    return item().more;
  }
};

// The run of this CTA, into each warp's walk; false when it has none.  All threads of the block (NT_ of them) call it.
template <int NT_>
TKB_DEVFN bool chunk_deal(const ChunkParams& p, ChunkWalk& w) {
  __shared__ long long s_sum[NT_ / 32], s_x;
  __shared__ int s_units[NT_ / 32], s_at[3];
  __shared__ ChunkSeq s_seq;
  const int tid = threadIdx.x, lane = lane_id(), wid = warp_id();
  const int per = (p.c.B + NT_ - 1) / NT_, b0 = min(tid * per, p.c.B), b1 = min(b0 + per, p.c.B);
  const int groups = p.c.Hkv * p.hb;
  // the costs of this thread's sequences, and their sums over the block
  ChunkSeq s;
  long long cost = 0, mine = 0, total = 0;
  int units = 0;
#pragma unroll 1
  for (int b = b0; b < b1; ++b) {
    s = chunk_seq(p, b);
    cost = chunk_seq_cost(p, s);
    mine += cost * groups;
    units = static_cast<int>(min(units + static_cast<long long>(s.units) * groups, 0xFFFFll));
  }
  long long upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += y;
  }
  units = __reduce_add_sync(0xffffffffu, units);
  if (lane == 31) {
    s_sum[wid] = upto;
    s_units[wid] = units;
  }
  __syncthreads();
  units = 0;
#pragma unroll 1
  for (int i = 0; i < NT_ / 32; ++i) {
    if (i == wid) upto += total;
    total += s_sum[i];
    units += s_units[i];
  }
  int ctas = gridDim.x;
  if (total < static_cast<long long>(ctas) * p.cost.least)
    ctas = min(ctas, max(units, (static_cast<int>(total) + p.cost.least - 1) / p.cost.least));
  const int c = blockIdx.x;
  if (c >= ctas) return false;
  // total * c / ctas
  const long long each = total / ctas;
  const int rest = static_cast<int>(total - each * ctas);
  const long long x0 = each * c + rest * c / ctas, x1 = each * (c + 1) + rest * (c + 1) / ctas;
  upto -= mine;
  if (upto <= x0 && x0 < upto + mine) {  // the run starts in one of this thread's sequences
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
      if (per > 1) {
        s = chunk_seq(p, b);
        cost = chunk_seq_cost(p, s);
      }
      if (x0 < upto + cost * groups) {
        int hg = 0;
#pragma unroll 1
        for (; x0 >= upto + cost; ++hg) upto += cost;
        int lo = 0, hi = s.units - 1;  // last unit that starts at x0 or before
#pragma unroll 1
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (upto + chunk_cost_before(p, s.base, mid) <= x0) lo = mid;
          else hi = mid - 1;
        }
        s_at[0] = b;
        s_at[1] = hg;
        s_at[2] = lo;
        s_x = upto + chunk_cost_before(p, s.base, lo);
        s_seq = s;
        break;
      }
      upto += cost * groups;
    }
  }
  __syncthreads();
  if (lane == 0) {
    w.b = s_at[0];
    w.hg = s_at[1];
    w.u = s_at[2];
    w.at = s_x;
    w.x0 = x0;
    w.x1 = x1;
    w.it[0].s = s_seq;
    w.k = 0;
  }
  __syncwarp();
  return true;
}

// What a CTA left in the workspace: a part of a unit that earlier CTAs began, whether it is the unit's last, and the
// first part of a unit that goes on in later ones.
enum ChunkSpan : int { SPAN_GOES_ON = 1, SPAN_ENDS = 2, SPAN_BEGINS = 4 };

// The (sequence row, query head) of row r of tile w of a unit, r = (t, g) in tokens and heads; false where there is none.
TKB_DEVFN bool chunk_row(const ChunkParams& p, int hg, int t0, int tokens, int w, int t, int g, int& tok, int& hq) {
  int h = hg;
  if (p.hb > 1) {
    h = hg / p.hb;
    g += (hg - h * p.hb) * p.gb;
  }
  tok = t0 + w * p.tt + t;
  hq = h * p.G + g;
  return t < p.tt && w * p.tt + t < tokens && g < p.G;
}

// ============================================================ 16-bit types: tcgen05
constexpr int kChunkThreads = 352;  // softmax 0-7, Q and K loads 8, products 9, V loads 10
template <int D>
struct ChunkCfg {
  static constexpr int TILE = 128 * D * 2;  // bytes of one 128-row x D tile
  static constexpr int SLAB = 128 * 128;    // bytes of one 64-column swizzle slab
  static constexpr int NST = D == 64 ? 4 : 2;  // stages of the K ring and of the V ring
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + 2 * TILE;
  static constexpr int OFF_V = OFF_K + NST * TILE;
  static constexpr int OFF_X = OFF_V + NST * TILE;       // 32 columns of the second warpgroup's O, [8][128] float4
  static constexpr int OFF_XML = OFF_X + 128 * 32 * 4;
  static constexpr int OFF_BAR = OFF_XML + 128 * 8;
  // q_full, q_empty, k_full[NST], k_empty[NST], v_full[NST], v_empty[NST], s_full[2], p_ready[2][2], o_done[2],
  // x_full, x_empty, drain
  static constexpr int NBAR = 2 + 4 * NST + 8 + 3;
  static constexpr int NMASK = 16;                       // page marks of the newest blocks (more than are in flight)
  static constexpr int OFF_MASK = OFF_BAR + NBAR * 8;
  static constexpr int OFF_WALK = (OFF_MASK + NMASK * 4 + 7) / 8 * 8;
  static constexpr int OFF_MISC = OFF_WALK + kChunkThreads / 32 * sizeof(ChunkWalk);
  static constexpr int SMEM = OFF_MISC + 16 + 1024;      // + slack for 1024-byte alignment
  static_assert(SMEM <= 232448, "tiles exceed 227 KB of shared memory");
  static constexpr uint32_t TM_S0 = 0, TM_S1 = 128, TM_O0 = 256, TM_O1 = 256 + D;
};

TKB_DEVFN void wait_ld16_dep(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// One block of the online softmax for this thread's query row: S from TMEM,
// slots from `lim` on and those of bad pages (bits of `there`, 16 slots each) masked, the
// running maximum raised when this block's exceeds it by more than 8
// (rescaling O in TMEM), P written over S in two halves, release(h) once half
// h is in TMEM.  P is rounded to the type (half a step; the row sum is that of
// the unrounded values): the error against 64 bits is 0.0021-0.0023 in bf16 where
// the output's own rounding is 0.0016-0.0017.  P in two 16-bit parts and a second
// product with V, in units of one tile alone, leave the output's rounding, but
// their instructions take 32 ragged sequences from 92 to 142 us, 8 x 3-6 tokens
// over 12-16 k from 101 to 141 and 64 single tokens from 87 to 143.
template <int D, bool BF16, typename Release>
TKB_DEVFN void chunk_softmax(uint32_t tS, uint32_t tO, float sl2, bool first, bool cut, int lim, unsigned there,
                             float& m_used, float& l, Release&& release) {
  uint32_t r0[32], r1[32], r2[32], r3[32];
  tmem_ld32(tS + 0, r0);
  tmem_ld32(tS + 32, r1);
  tmem_ld32(tS + 64, r2);
  tmem_ld32(tS + 96, r3);
  wait_ld_dep(r0);
  wait_ld_dep(r1);
  wait_ld_dep(r2);
  wait_ld_dep(r3);
  float sv[128];
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    sv[i] = __uint_as_float(r0[i]);
    sv[32 + i] = __uint_as_float(r1[i]);
    sv[64 + i] = __uint_as_float(r2[i]);
    sv[96 + i] = __uint_as_float(r3[i]);
  }
  if (cut) {
#pragma unroll
    for (int c = 0; c < 128; ++c)
      if (c >= lim || !(there >> (c >> 4) & 1)) sv[c] = -INFINITY;
  }
  float mx0 = sv[0], mx1 = sv[1], mx2 = sv[2], mx3 = sv[3];
#pragma unroll
  for (int c = 4; c < 124; c += 8) {
    mx0 = fmax3(mx0, sv[c], sv[c + 1]);
    mx1 = fmax3(mx1, sv[c + 2], sv[c + 3]);
    mx2 = fmax3(mx2, sv[c + 4], sv[c + 5]);
    mx3 = fmax3(mx3, sv[c + 6], sv[c + 7]);
  }
  mx0 = fmax3(mx0, sv[124], sv[125]);
  mx1 = fmax3(mx1, sv[126], sv[127]);
  // m is kept UP below the maximum, so that f16 weights, at most 2^(8 + UP), lie as far as they can above the type's
  // smallest value, 2^-24: what is rounded to 0 is below 2^-31 of the largest
  constexpr float UP = BF16 ? 0.f : 7.f;
  const float mx = fmaf(fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)), sl2, -UP);
  float resc = 1.f;
  bool raised = false;
  if (first) {
    m_used = mx;
  } else if (mx > m_used + 8.0f) {  // from -inf too: the O so far is then a sum of zeros
    resc = ex2(m_used - mx);
    l *= resc;
    m_used = mx;
    raised = true;
  }
  const float base = m_used == -INFINITY ? 0.f : -m_used;
  const uint64_t sl2x2 = f2(sl2, sl2), nmx2 = f2(base, base);
  uint32_t pk0[32], pk1[32];
  uint64_t ls0 = f2(0.f, 0.f), ls1 = f2(0.f, 0.f);
  auto exp_pair = [&](int from, int i, uint32_t& pk, uint64_t& ls) {
    float x0, x1, a, c;
    f2_split(fma_f2(f2(sv[from + 2 * i], sv[from + 2 * i + 1]), sl2x2, nmx2), x0, x1);
    a = ex2(x0);
    c = ex2(x1);
    ls = add_f2(ls, f2(a, c));
    pk = pack2_int<BF16>(a, c);
  };
#pragma unroll
  for (int i = 0; i < 32; ++i) exp_pair(0, i, pk0[i], (i & 1) ? ls1 : ls0);
  if (__any_sync(0xffffffffu, raised)) {  // warp-collective, as the prompt's own attention does it
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t o[32];
      tmem_ld32(tO + c * 32, o);
      wait_ld_dep(o);
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * resc);
      tmem_st32(tO + c * 32, o);
    }
  }
  tmem_st32(tS + 0, pk0);
  tmem_wait_st();
  tc_fence_before();
  release(0);
  if (cut && __all_sync(0xffffffffu, lim <= 64)) {  // nothing of the second half is seen
#pragma unroll
    for (int i = 0; i < 32; ++i) pk1[i] = 0u;
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) exp_pair(64, i, pk1[i], (i & 1) ? ls1 : ls0);
  }
  {
    float a0, a1, b0, b1;
    f2_split(ls0, a0, a1);
    f2_split(ls1, b0, b1);
    l += (a0 + b0) + (a1 + b1);
  }
  tmem_st32(tS + 32, pk1);
  tmem_wait_st();
  tc_fence_before();
  release(1);
}

// Where a finished row of an item goes: out, or a part in the workspace.
struct ChunkSink {
  bool part;
  long long slot;  // part: index of (CTA, which, tile) * 128 + row
  float inv;       // out: 1 / l, 0 for a row that sees nothing
  uint16_t* out;   // out: column 0 of the row's head
};
template <int D, bool BF16>
TKB_DEVFN void chunk_put4(const ChunkParams& p, const ChunkSink& k, int col4, float a, float b, float c, float d) {
  if (k.part) {
    // [tile][D / 4][128]: the rows of a warp side by side
    p.part[(k.slot >> 7) * (D / 4) * 128 + col4 * 128 + (k.slot & 127)] = make_float4(a, b, c, d);
  } else {
    uint2 v = make_uint2(0u, 0u);
    if (k.inv != 0.f) v = make_uint2(pack2<BF16>(a * k.inv, b * k.inv), pack2<BF16>(c * k.inv, d * k.inv));
    *reinterpret_cast<uint2*>(k.out + col4 * 4) = v;
  }
}

// A value of V that is not finite, in a slot that some rows of a tile see and
// others do not, spoils the products of those others too (0 * inf).  A CTA that
// meets a row whose O is not finite though its sum is, and which has slots of its
// item behind its last one, walks its run a second time, with care: in slots that
// not all rows of a unit see, such values become 0 in shared memory before their
// products, and once a row is written, those that it does see are added to it.
// (2 x 1.7 k tokens over 16 k, such a value near each end: 1.72 -> 3.55 ms.  No
// wait of the run, bounded as they are, has to cover more than a block of it.)
// 128 threads: the values of slots from .. upto - 1 of a stage of V.
template <int D, bool BF16>
__noinline__ __device__ void chunk_take_out(uint8_t* stage, int from, int upto, int r) {
  constexpr uint32_t EXP = BF16 ? 0x7f80u : 0x7c00u;  // all ones: an infinity or NaN
  for (int i = from * 8 + r; i < upto * 8; i += 128)
#pragma unroll 1
    for (int x = 0; x < D / 64; ++x) {
      uint32_t* at = reinterpret_cast<uint32_t*>(stage + x * 128 * 128 + i * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t v = at[e];
        uint32_t keep = 0u;
        if ((v & EXP) != EXP) keep |= 0xffffu;
        if ((v >> 16 & EXP) != EXP) keep |= 0xffff0000u;
        if (~keep) at[e] = v & keep;
      }
    }
}
// Whole warps, a row a lane: the values taken out of blocks j0, j0 + step, ... below slot `last`, from slot `from` on.
template <int D, bool BF16>
__noinline__ __device__ void chunk_add_back(const ChunkParams& p, int b, int h, int j0, int step, int from, int last, int lim,
                                            int row, int hq, float m, const ChunkSink& sink) {
  constexpr int E = D / 32;
  const tkb_kv_cache& c = p.c;
  const int lane = lane_id();
  using U = typename std::conditional<E == 4, uint2, uint32_t>::type;
  auto load = [&](const void* pool, long long at, float (&f)[E]) {
    const U u = *reinterpret_cast<const U*>(static_cast<const uint16_t*>(pool) + at + lane * E);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      const float2 x = unpack2<BF16>(w[e]);
      f[2 * e] = x.x;
      f[2 * e + 1] = x.y;
    }
  };
  __syncwarp();  // the rows' other lanes have written them
#pragma unroll 1
  for (int j = max(from, j0 * kChunkBlock); j < last; ++j) {
    if ((j / kChunkBlock - j0) % step) continue;  // the other warpgroup's
    const int pg = c.block_table[static_cast<long long>(b) * c.max_pages + j / c.page_size];
    if (static_cast<unsigned>(pg) >= static_cast<unsigned>(c.n_pages)) continue;
    const long long at = page_offset(c, pg, h) + static_cast<long long>(j % c.page_size) * D;
    float k[E], v[E];
    load(c.v, at, v);
    bool odd = false;
#pragma unroll
    for (int e = 0; e < E; ++e) odd |= !(fabsf(v[e]) < INFINITY);
    if (!__any_sync(0xffffffffu, odd)) continue;
    load(c.k, at, k);
#pragma unroll 1
    for (unsigned todo = __ballot_sync(0xffffffffu, lim > j); todo; todo &= todo - 1) {
      const int src = __ffs(todo) - 1, rr = __shfl_sync(0xffffffffu, row, src), rh = __shfl_sync(0xffffffffu, hq, src);
      const float rm = __shfl_sync(0xffffffffu, m, src), inv = __shfl_sync(0xffffffffu, sink.inv, src);
      const long long slot = __shfl_sync(0xffffffffu, sink.slot, src);
      float q[E], s = 0.f;
      load(p.q, rr * p.q_stride + static_cast<long long>(rh) * D, q);
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(q[e], k[e], s);
      const float pr = ex2(fmaf(warp_sum(s), p.scale_log2, rm == -INFINITY ? 0.f : -rm));
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (fabsf(v[e]) < INFINITY) continue;
        const int col = lane * E + e;
        if (sink.part) {
          float* o = reinterpret_cast<float*>(p.part + (slot >> 7) * (D / 4) * 128 + (col >> 2) * 128 + (slot & 127)) + (col & 3);
          *o = fmaf(pr, v[e], *o);
        } else {
          uint16_t* o = static_cast<uint16_t*>(p.out) + rr * p.out_stride + static_cast<long long>(rh) * D + col;
          *o = static_cast<uint16_t>(pack2<BF16>(fmaf(pr * inv, v[e], unpack2<BF16>(*o).x), 0.f));
        }
      }
    }
  }
}

// Where things lie in shared memory.
TKB_DEVFN uint8_t* chunk_smem() {
  extern __shared__ uint8_t smem_raw[];
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
}
template <int D>
struct ChunkShared {
  using C = ChunkCfg<D>;
  uint64_t *q_full, *q_empty, *k_full, *k_empty, *v_full, *v_empty, *s_full, *p_ready, *o_done, *x_full, *x_empty, *mma_drain;
  uint32_t *marks, *tmem_slot;
  volatile int *abort_flag, *again_flag;
  ChunkWalk* walk;
  TKB_DEVFN explicit ChunkShared(uint8_t* smem) {
    q_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    q_empty = q_full + 1;
    k_full = q_full + 2;
    k_empty = k_full + C::NST;
    v_full = k_empty + C::NST;
    v_empty = v_full + C::NST;
    s_full = v_empty + C::NST;
    p_ready = s_full + 2;  // [w][half]
    o_done = p_ready + 4;
    x_full = o_done + 2;
    x_empty = x_full + 1;
    mma_drain = x_empty + 1;
    marks = reinterpret_cast<uint32_t*>(smem + C::OFF_MASK);
    tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
    abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
    again_flag = abort_flag + 1;
    walk = reinterpret_cast<ChunkWalk*>(smem + C::OFF_WALK) + warp_id();
  }
};

// The roles of a CTA over its run.  CAREFUL: the second walk, which counts on from the first.
template <int D, bool BF16, bool CAREFUL>
TKB_DEVFN void chunk_tc_run(const ChunkParams& p, uint8_t* smem, uint32_t tmem, bool any) {
  using C = ChunkCfg<D>;
  const uint32_t sbase = smem_u32(smem);
  const ChunkShared<D> sh(smem);
  uint64_t *const q_full = sh.q_full, *const q_empty = sh.q_empty, *const k_full = sh.k_full, *const k_empty = sh.k_empty,
           *const v_full = sh.v_full, *const v_empty = sh.v_empty, *const s_full = sh.s_full, *const p_ready = sh.p_ready,
           *const o_done = sh.o_done, *const x_full = sh.x_full, *const x_empty = sh.x_empty, *const mma_drain = sh.mma_drain;
  uint32_t* const marks = sh.marks;
  volatile int *const abort_flag = sh.abort_flag, *const again_flag = sh.again_flag;
  ChunkWalk& walk = *sh.walk;
  const int warp = warp_id(), lane = lane_id();
  auto counted = [&](int i) { return CAREFUL ? walk.count[i] : 0; };
  if (!any) {
    if (threadIdx.x == 0) p.span[blockIdx.x] = make_int4(0, 0, 0, 0);
  } else if (warp == 8 || warp == 10) {
    // ------------------------------------------------------------ TMA producers
    // A lane issues one box: `gran` slots of one 64-column slab of K or V.  Two warps, because boxes of 16 slots are 16 to
    // 32 of these instructions a block, some 0.1 us each from one warp.
    const bool keys = warp == 8;
    uint64_t* full = keys ? k_full : v_full;
    uint64_t* empty = keys ? k_empty : v_empty;
    const CUtensorMap* map = keys ? &p.tmK : &p.tmV;
    uint8_t* ring = smem + (keys ? C::OFF_K : C::OFF_V);
    const int boxes = kChunkBlock / p.gran, nl = boxes * (D / 64);
    const int gi = lane % boxes, hh = lane / boxes;
    const int box_rows = p.gran;
    const uint32_t q_bytes = static_cast<uint32_t>(p.gb) * p.tt * D * 2;
    int nq = counted(0), nb = counted(1);  // loads issued
    bool ok = true;
    walk.ahead(p);
    while (ok && walk.next()) {
      const ChunkItem& it = walk.item();
      const ChunkSeq& s = it.s;
      const int h = it.hg / p.hb, hq0 = h * p.G + (it.hg % p.hb) * p.gb, jb = it.jb, je = it.je;
      const bool pair = it.pair(p);
      // read once by a unit alone, or by the units that follow too
      const uint64_t pol_q = policy_evict_first(), pol_kv = s.units > 1 ? policy_evict_last() : policy_evict_first();
      const int32_t* table = p.c.block_table + static_cast<long long>(it.b) * p.c.max_pages;
      // this lane's page in block j: beyond the pool (the box is then zeros) where there is none
      auto page_in = [&](int j, bool& bad) {
        const int slot = j * kChunkBlock + gi * box_rows;
        bad = false;
        if (lane >= nl || slot >= s.held) return p.c.n_pages;
        const int pg = __ldg(table + slot / p.c.page_size);
        bad = static_cast<unsigned>(pg) >= static_cast<unsigned>(p.c.n_pages);
        return bad ? p.c.n_pages : pg;
      };
      bool bad;
      int page = page_in(jb, bad);
      if (keys) {
        if (!(ok = mbar_wait_warp(q_empty, (nq & 1) ^ 1, abort_flag))) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(q_full, (pair ? 2 : 1) * q_bytes);
          for (int w = 0; w < (pair ? 2 : 1); ++w)
#pragma unroll
            for (int x = 0; x < D / 64; ++x)
              tma_load_3d(smem + C::OFF_Q + w * C::TILE + x * C::SLAB, &p.tmQ, q_full, x * 64, hq0,
                          s.first + it.t0 + w * p.tt, pol_q);
        }
        ++nq;
      }
      walk.ahead(p);
      for (int j = jb; j < je; ++j) {
        bool bad_next = false;
        int next = 0;
        if (j + 1 < je) next = page_in(j + 1, bad_next);
        const int in_head = (j * kChunkBlock + gi * box_rows) % p.c.page_size + h * p.c.page_size;
        const int stage = nb % C::NST;
        if (!(ok = mbar_wait_warp(&empty[stage], ((nb / C::NST) & 1) ^ 1, abort_flag))) break;
        if (keys) {
          // bits of the 16-slot groups that lie in bad pages
          const unsigned lost = __reduce_or_sync(0xffffffffu, bad ? ((1u << (box_rows / 16)) - 1) << (gi * box_rows / 16) : 0u);
          if (lane == 0) {
            if (lost) atomicOr(&g_device_error, ERR_BAD_INDEX);
            marks[nb % C::NMASK] = ~lost;
          }
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[stage], C::TILE);
        __syncwarp();
        if (lane < nl)
          tma_load_3d(ring + stage * C::TILE + hh * C::SLAB + gi * box_rows * 128, map, &full[stage], hh * 64, in_head, page,
                      pol_kv);
        ++nb;
        page = next;
        bad = bad_next;
      }
    }
    __syncwarp();
    if (!CAREFUL && lane == 0) {
      walk.count[0] = nq;
      walk.count[1] = nb;
    }
    if (*abort_flag) {
      // Let every copy this CTA started land before the CTA exits.
      volatile int never = 0;
      if (nq) mbar_wait(q_full, (nq - 1) & 1, &never);
      for (int i = max(0, nb - C::NST); i < nb; ++i) mbar_wait(&full[i % C::NST], (i / C::NST) & 1, &never);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {  // steps its walk alone
      constexpr uint32_t idS = idesc_f16kind(128, 128, BF16, false, false);
      constexpr uint32_t idO = idesc_f16kind(128, D, BF16, false, true);
      const uint32_t sQ = sbase + C::OFF_Q, sK = sbase + C::OFF_K, sV = sbase + C::OFF_V;
      auto issue_S = [&](int w, int tile, int stage) {  // S of warpgroup w: its tile's queries, the stage's keys
        const uint32_t qa = sQ + tile * C::TILE, ka = sK + stage * C::TILE;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * C::SLAB + (kk & 3) * 32;
          umma_ss(tmem + (w ? C::TM_S1 : C::TM_S0), sdesc_sw128(qa + off, 16, 1024),
                  sdesc_sw128(ka + off, 16, 1024), idS, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[w]);
      };
      auto issue_PV = [&](int w, int stage, int half, bool acc) {
        const uint32_t va = sV + stage * C::TILE;
        const uint32_t tP = tmem + (w ? C::TM_S1 : C::TM_S0);
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4) {
          const int kk = half * 4 + k4;
          umma_ts(tmem + (w ? C::TM_O1 : C::TM_O0), tP + kk * 8, sdesc_sw128(va + kk * 2048, C::SLAB, 1024), idO,
                  (acc || kk > 0) ? 1u : 0u);
        }
      };
      int nq = counted(0), nk = counted(1), nv = counted(2);  // Q tiles, K and V blocks met so far
      int np[2] = {counted(3), counted(4)};  // blocks of each warpgroup whose P has been used
      bool ok = true;
      auto wait_k = [&]() {
        if (!(ok = mbar_wait(&k_full[nk % C::NST], (nk / C::NST) & 1, abort_flag))) return false;
        tc_fence_after();
        return true;
      };
      auto half_PV = [&](int w, int half, bool acc) {
        if (!(ok = mbar_wait(&p_ready[2 * w + half], np[w] & 1, abort_flag))) return false;
        tc_fence_after();
        issue_PV(w, nv % C::NST, half, acc);
        return true;
      };
      for (walk.step(p), ++walk.k; ok && walk.item().more; walk.step(p), ++walk.k) {
        const ChunkItem& it = walk.item();
        if (!(ok = mbar_wait(q_full, nq & 1, abort_flag))) break;
        ++nq;
        tc_fence_after();
        const int jb = it.jb, je = it.je;
        if (it.pair(p)) {
          // both warpgroups meet the same blocks, each with its own tile; the first tile's may end earlier
          const int end[2] = {min(je, it.nb0), je};
          if (!wait_k()) break;
          for (int w = 0; w < 2; ++w)
            if (jb < end[w]) issue_S(w, w, nk % C::NST);
          umma_commit(&k_empty[nk % C::NST]);
          ++nk;
          if (jb + 1 == je) umma_commit(q_empty);
          for (int j = jb; ok && j < je; ++j) {
            if (!(ok = mbar_wait(&v_full[nv % C::NST], (nv / C::NST) & 1, abort_flag))) break;
            bool k_next = false;
            for (int w = 0; w < 2 && ok; ++w) {
              if (j >= end[w]) continue;
              if (!half_PV(w, 0, j > jb) || !half_PV(w, 1, true)) break;
              ++np[w];
              if (j + 1 == end[w]) umma_commit(&o_done[w]);
              if (j + 1 < end[w]) {
                if (!k_next && !wait_k()) break;
                k_next = true;
                issue_S(w, w, nk % C::NST);
              }
            }
            if (!ok) break;
            umma_commit(&v_empty[nv % C::NST]);
            ++nv;
            if (k_next) {
              umma_commit(&k_empty[nk % C::NST]);
              ++nk;
              if (j + 2 == je) umma_commit(q_empty);
            }
          }
        } else {
          // the warpgroups take the blocks of the one tile in turn
          const int n = je - jb;
          for (int i = 0; i < min(n, 2); ++i) {
            if (!wait_k()) break;
            issue_S(i, 0, nk % C::NST);
            umma_commit(&k_empty[nk % C::NST]);
            ++nk;
          }
          if (ok && n <= 2) umma_commit(q_empty);
          for (int i = 0; ok && i < n; ++i) {
            const int w = i & 1;
            if (!(ok = mbar_wait(&v_full[nv % C::NST], (nv / C::NST) & 1, abort_flag))) break;
            if (!half_PV(w, 0, i > 1) || !half_PV(w, 1, true)) break;
            ++np[w];
            umma_commit(&v_empty[nv % C::NST]);
            ++nv;
            if (i + 2 >= n) umma_commit(&o_done[w]);
            if (i + 2 < n) {
              if (!wait_k()) break;
              issue_S(w, 0, nk % C::NST);
              umma_commit(&k_empty[nk % C::NST]);
              ++nk;
              if (i + 3 == n) umma_commit(q_empty);
            }
          }
        }
      }
      if (!CAREFUL) {
        walk.count[0] = nq;
        walk.count[1] = nk;
        walk.count[2] = nv;
        walk.count[3] = np[0];
        walk.count[4] = np[1];
      }
      if (!ok) {
        // Make sure no MMA is still running when TMEM is released.
        volatile int never = 0;
        umma_commit(mma_drain);
        mbar_wait(mma_drain, 0, &never);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax warpgroups
    const int w = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_off + (w ? C::TM_S1 : C::TM_S0);
    const uint32_t tO = tmem + lane_off + (w ? C::TM_O1 : C::TM_O0);
    float4* xo = reinterpret_cast<float4*>(smem + C::OFF_X);
    float2* xml = reinterpret_cast<float2*>(smem + C::OFF_XML);
    const float sl2 = p.scale_log2;
    // blocks of this warpgroup, items with blocks of it, blocks of the CTA, exchanges
    int ns = counted(0), no = counted(1), nb = counted(2), nx = counted(3);
    int flags = 0, span_b = 0, span_hg = 0, span_u = 0;
    bool ok = true;
    const int row_t = r / p.gb, row_g = r - row_t * p.gb;
    walk.ahead(p);
    while (ok && walk.next()) {
      const ChunkItem& it = walk.item();
      const ChunkSeq& s = it.s;
      const bool pair = it.pair(p);
      const int tile = pair ? w : 0;
      int tok, hq;
      const bool valid = chunk_row(p, it.hg, it.t0, it.tokens, tile, row_t, row_g, tok, hq);
      const int lim = valid ? min(max(s.base + tok + 1, 0), s.held) : 0;
      const bool busy = __any_sync(0xffffffffu, valid);  // a warp without rows leaves its P as it is: nobody reads its O
      const int tile_lim = min(max(s.base + it.t0 + tile * p.tt + 1, 0), s.held);  // what the tile's first row sees
      const int step = pair ? 1 : 2, j0 = it.jb + (pair ? 0 : w), end = pair && w == 0 ? min(it.je, it.nb0) : it.je;
      float m = -INFINITY, l = 0.f;
      for (int j = j0; j < end; j += step) {
        const int at = j * kChunkBlock, nth = nb + j - it.jb;
        if (!(ok = mbar_wait_warp(&s_full[w], ns & 1, abort_flag))) break;
        tc_fence_after();
        const int all_see = CAREFUL ? min(max(s.base + it.t0 + 1, 0), s.held) : s.held;  // what the unit's first row sees
        if (at + kChunkBlock > all_see) {
          // slots of the last page behind the sequence's end may hold anything, and 0 * NaN is NaN: V there becomes 0
          const int stage = nth % C::NST;
          if (!(ok = mbar_wait_warp(&v_full[stage], (nth / C::NST) & 1, abort_flag))) break;
          const int from = max(s.held - at, 0);
          if constexpr (CAREFUL)
            chunk_take_out<D, BF16>(smem + C::OFF_V + stage * C::TILE, max(all_see - at, 0), min(from, kChunkBlock), r);
          for (int i = from * 8 + r; i < kChunkBlock * 8; i += 128)
#pragma unroll
            for (int x = 0; x < D / 64; ++x)
              *reinterpret_cast<uint4*>(smem + C::OFF_V + stage * C::TILE + x * C::SLAB + i * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
        }
        const unsigned there = *reinterpret_cast<volatile uint32_t*>(&marks[nth % C::NMASK]);
        auto release = [&](int half) { mbar_arrive(&p_ready[2 * w + half]); };
        if (busy) {
          chunk_softmax<D, BF16>(tS, tO, sl2, j == j0, at + kChunkBlock > tile_lim || there != ~0u, lim - at, there, m, l,
                                 release);
        } else {
          release(0);
          release(1);
        }
        ++ns;
      }
      if (!ok) break;
      nb += it.je - it.jb;
      walk.ahead(p);  // while the last products run
      const bool has = j0 < end;
      if (has) {
        if (!(ok = mbar_wait_warp(&o_done[w], no & 1, abort_flag))) break;
        ++no;
        tc_fence_after();
      }
      // ---- the warpgroups' halves of a whole unit of one tile meet: the second hands over its m, l and O, 32 columns
      // at a time.  (Of a part, each leaves its own half in the workspace.)
      const bool whole = it.whole(), meet = !pair && whole && it.je - it.jb > 1;
      if (!pair && w == 1 && whole) {
        if (meet) {
          xml[r] = make_float2(m, l);
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            if (!(ok = mbar_wait_warp(x_empty, (nx & 1) ^ 1, abort_flag))) break;
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            wait_ld_dep(o);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              xo[i * 128 + r] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                            __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
            mbar_arrive(x_full);
            ++nx;
          }
        }
        continue;
      }
      // ---- the tile's rows go out (loops that are not unrolled: this code runs once a unit, from a cold instruction cache)
      ChunkSink sink;
      sink.part = !whole;
      const int which = it.jb > 0 ? 0 : 1;
      sink.slot = ((2ll * blockIdx.x + which) * 2 + w) * 128 + r;
      if (sink.part) {
        flags |= which ? SPAN_BEGINS : SPAN_GOES_ON | (it.je == it.nb1 ? SPAN_ENDS : 0);
        if (which) {
          span_b = it.b;
          span_hg = it.hg;
          span_u = it.u;
        }
      }
      const int row = s.first + tok;
      sink.out = valid ? static_cast<uint16_t*>(p.out) + row * p.out_stride + static_cast<long long>(hq) * D : nullptr;
      // two lanes write 32 bytes of a row: where this lane's 16 bytes of its pair's two rows go
      uint16_t* rows2[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        rows2[i] = reinterpret_cast<uint16_t*>(
            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(sink.out), (lane & ~1) + i));
        if (rows2[i]) rows2[i] += (lane & 1) * 8;
      }
      float4* part = p.part + (sink.slot >> 7) * (D / 4) * 128 + r;
      float f0 = 1.f, f1 = 0.f, zero = 0.f;
      bool sees0 = true, sees1 = false;  // a half that saw nothing has an O of masked values alone
#pragma unroll 1
      for (int c = 0; c < D / 16; ++c) {
        if (meet && !(c & 1)) {  // the other's columns
          if (!(ok = mbar_wait_warp(x_full, nx & 1, abort_flag))) break;
          if (c == 0) {
            const float2 ml = xml[r];
            const float mm = fmaxf(m, ml.x);
            sees0 = m != -INFINITY;
            sees1 = ml.x != -INFINITY;
            f0 = sees0 ? ex2(m - mm) : 0.f;
            f1 = sees1 ? ex2(ml.x - mm) : 0.f;
            l = f0 * l + f1 * ml.y;
            m = m != m ? m : mm;
          }
        }
        if (c == 0) {
          sink.inv = l == 0.f ? 0.f : 1.f / l;
          if (valid) {
            if (sink.part) p.part_ml[sink.slot] = make_float2(m, l);
            else if (p.lse) p.lse[static_cast<long long>(row) * p.Hq + hq] = (m + lg2(l)) * 0.69314718055994531f;
          }
          if (!has) break;  // a tile whose blocks lie before the run's
        }
        uint32_t o[16];
        tmem_ld16(tO + c * 16, o);
        wait_ld16_dep(o);
        if (meet) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 x = xo[((c & 1) * 4 + i) * 128 + r];
            const float b[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[4 * i + e] = __float_as_uint((sees0 ? f0 * __uint_as_float(o[4 * i + e]) : 0.f) + (sees1 ? f1 * b[e] : 0.f));
          }
          if (c & 1) {
            mbar_arrive(x_empty);
            ++nx;
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) zero = fmaf(__uint_as_float(o[i]), 0.f, zero);  // NaN once a value is not finite
        if (sink.part) {
          if (valid) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              part[(c * 4 + i) * 128] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                    __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
          }
        } else {
          uint32_t v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[i] = sink.inv == 0.f ? 0u : pack2<BF16>(__uint_as_float(o[2 * i]) * sink.inv, __uint_as_float(o[2 * i + 1]) * sink.inv);
          const bool odd = lane & 1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // lane i of the pair: 16 bytes i of both rows
            const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[4 + i], 1);
            v[i] = odd ? got : v[i];
            v[4 + i] = odd ? v[4 + i] : got;
          }
          if (rows2[0]) *reinterpret_cast<uint4*>(rows2[0] + c * 16) = make_uint4(v[0], v[1], v[2], v[3]);
          if (rows2[1]) *reinterpret_cast<uint4*>(rows2[1] + c * 16) = make_uint4(v[4], v[5], v[6], v[7]);
        }
      }
      if (!ok) break;
      const int last = min(end * kChunkBlock, s.held);
      if constexpr (CAREFUL) {
        chunk_add_back<D, BF16>(p, it.b, it.hg / p.hb, meet ? it.jb : j0, meet ? 1 : step,
                                min(max(s.base + it.t0 + 1, 0), s.held), last, lim, row, hq, m, sink);
      } else if (has && !(zero == 0.f) && valid && l > 0.f && lim < last) {
        *again_flag = 1;  // O is not finite though l is
      }
    }
    __syncwarp();
    if (!CAREFUL && lane == 0) {
      walk.count[0] = ns;
      walk.count[1] = no;
      walk.count[2] = nb;
      walk.count[3] = nx;
    }
    if (threadIdx.x == 0) p.span[blockIdx.x] = make_int4(ok ? flags : 0, span_b, span_hg, span_u);
  }
}
template <int D, bool BF16>
__noinline__ __device__ void chunk_tc_again(const ChunkParams& p) {
  uint8_t* smem = chunk_smem();
  const ChunkShared<D> sh(smem);
  const bool any = chunk_deal<kChunkThreads>(p, *sh.walk);
  chunk_tc_run<D, BF16, true>(p, smem, *sh.tmem_slot, any);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kChunkThreads, 1) chunk_tc_kernel(const __grid_constant__ ChunkParams p) {
  using C = ChunkCfg<D>;
  uint8_t* smem = chunk_smem();
  const ChunkShared<D> sh(smem);
  const int warp = warp_id();

  if (threadIdx.x == 0) {
    for (uint64_t* x : {sh.q_full, sh.q_empty, sh.mma_drain}) mbar_init(x, 1);
    for (int s = 0; s < C::NST; ++s)
      for (uint64_t* x : {sh.k_full, sh.k_empty, sh.v_full, sh.v_empty}) mbar_init(x + s, 1);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&sh.s_full[w], 1);
      mbar_init(&sh.p_ready[2 * w], 128);
      mbar_init(&sh.p_ready[2 * w + 1], 128);
      mbar_init(&sh.o_done[w], 1);
    }
    mbar_init(sh.x_full, 128);
    mbar_init(sh.x_empty, 128);
    *sh.abort_flag = 0;
    *sh.again_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&p.tmQ);
    prefetch_tmap(&p.tmK);
    prefetch_tmap(&p.tmV);
  }
  if (warp == 9) {
    tmem_alloc(sh.tmem_slot, 512);
    tmem_relinquish();
  }
  grid_wait();
  grid_go();
  const bool any = chunk_deal<kChunkThreads>(p, *sh.walk);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  chunk_tc_run<D, BF16, false>(p, smem, *sh.tmem_slot, any);

  tc_fence_before();
  __syncthreads();
  if (*sh.again_flag && !*sh.abort_flag) {
    tc_fence_after();
    chunk_tc_again<D, BF16>(p);
    tc_fence_before();
    __syncthreads();
  }
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(*sh.tmem_slot, 512);
  }
}

// Joins the parts of units that span CTAs: the block of CTA c takes the unit
// that begins there and goes on behind it, with the parts of the CTAs that
// follow up to the one that ends it, in their order; of a unit of one tile each
// CTA has left two, its warpgroups'.  A thread has one row and 32 columns;
// blockIdx.y is tile and column group.
template <int D, typename T>
__global__ void __launch_bounds__(128) chunk_join_kernel(const __grid_constant__ ChunkParams p) {
  __shared__ int s_part[kChunkGrid], s_count[4], s_end;
  grid_wait();
  grid_go();
  const int c = blockIdx.x, w = blockIdx.y / (D / 32), cg = blockIdx.y % (D / 32), r = threadIdx.x, lane = lane_id();
  const int4 span = p.span[c];
  if (!(span.x & SPAN_BEGINS)) return;
  if (r == 0) s_end = gridDim.x - 1;
  __syncthreads();
  const ChunkSeq s = chunk_seq(p, span.y);
  const int t0 = span.w * 2 * p.tt, tokens = min(2 * p.tt, s.n - t0);
  const bool pair = tokens > p.tt;
  if (!pair && w) return;
  int parts = 0;  // the list of parts, 128 CTAs at a time up to the one that ends the unit
#pragma unroll 1
  for (int x0 = c; x0 < gridDim.x; x0 += 128) {
    const int x = x0 + r;
    const int flags = x == c || x >= gridDim.x ? 0 : p.span[x].x;
    if ((flags & (SPAN_GOES_ON | SPAN_ENDS)) == (SPAN_GOES_ON | SPAN_ENDS)) atomicMin(&s_end, x);
    __syncthreads();
    const bool mine = x == c || (x <= s_end && flags & SPAN_GOES_ON);
    const unsigned there = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) s_count[warp_id()] = __popc(there);
    __syncthreads();
    int at = parts + __popc(there & ((1u << lane) - 1));
    for (int i = 0; i < 4; ++i) {
      if (i < warp_id()) at += s_count[i];
      parts += s_count[i];
    }
    if (mine) s_part[at] = 2 * x + (x == c);
    __syncthreads();
    if (s_end < x0 + 128) break;
  }
  int tok, hq;
  if (!chunk_row(p, span.z, t0, tokens, w, r / p.gb, r % p.gb, tok, hq)) return;
  // part i of this row: of a pair its own tile's, else both warpgroups' in turn
  const int n = pair ? parts : 2 * parts;
  auto slot_of = [&](int i) { return pair ? 2ll * s_part[i] + w : 2ll * s_part[i >> 1] + (i & 1); };
  float m = -INFINITY;
  bool nan = false;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float x = p.part_ml[slot_of(i) * 128 + r].x;
    nan |= x != x;
    m = fmaxf(m, x);
  }
  if (nan) m = NAN;
  float l = 0.f, o[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) o[i] = 0.f;
#pragma unroll 2
  for (int k = 0; k < n; ++k) {
    const long long slot = slot_of(k);
    const float2 ml = p.part_ml[slot * 128 + r];
    const float4* part = p.part + slot * (D / 4) * 128 + cg * 8 * 128 + r;
    const bool sees = ml.x != -INFINITY;  // else its O is of masked values alone, or not written
    const float f = sees ? ex2(ml.x - m) : 0.f;
    l = fmaf(f, ml.y, l);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 v = sees ? part[i * 128] : make_float4(0.f, 0.f, 0.f, 0.f);
      o[4 * i] = fmaf(f, v.x, o[4 * i]);
      o[4 * i + 1] = fmaf(f, v.y, o[4 * i + 1]);
      o[4 * i + 2] = fmaf(f, v.z, o[4 * i + 2]);
      o[4 * i + 3] = fmaf(f, v.w, o[4 * i + 3]);
    }
  }
  const long long row = s.first + tok;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = static_cast<T*>(p.out) + row * p.out_stride + static_cast<long long>(hq) * D + cg * 32;
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = l == 0.f ? 0.f : o[i + e] * inv;
    stv<T, 8>(out + i, v);
  }
  if (p.lse && cg == 0) p.lse[row * p.Hq + hq] = (m + lg2(l)) * 0.69314718055994531f;
}

// ============================================================ fp32
// The same units and parts on FMA instructions, two at a time (f32x2): a CTA of
// 256 threads holds up to 128 packed rows (two tiles of 64) against 64 slots.
// Thread (tr, tc) of 16 x 16 has rows tr + 16 i, i < MR, and slots tc + 16 e of the scores,
// and columns 4 tc .. 4 tc + 3 of every 64 of the output, so that a row's
// scores, weights and sums stay in one half of a warp.  MR follows the unit's
// rows: with few of them the reads of K and V from shared memory are most of it.
// 8 sequences of 2-4 k, 8 kv heads of 128: 4 tokens x 2 heads 174 us (MR 1; 294 with
// 4, 521 with 8), 30 x 2 454 us (MR 4; 8: 782).
template <int D>
struct ChunkF32 {
  static constexpr int TS = 64;                            // slots at a time
  static constexpr int KS = D + 4, PS = TS + 4;            // floats from row to row: neighbours in different banks
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + 128 * KS * 4;
  static constexpr int OFF_V = OFF_K + TS * KS * 4;
  static constexpr int OFF_P = OFF_V + TS * D * 4;
  static constexpr int OFF_WALK = OFF_P + 128 * PS * 4;
  static constexpr int OFF_AT = OFF_WALK + 8 * sizeof(ChunkWalk);  // [2][TS] element offsets of the slots, -1 for none
  static constexpr int SMEM = OFF_AT + 2 * TS * 8;
  static_assert(SMEM <= 232448 && sizeof(ChunkWalk) % 8 == 0, "shared memory");
};

// The blocks of one item for MR rows a thread.
template <int D, int MR>
__noinline__ __device__ void chunk_f32_item(const ChunkParams& p, const ChunkItem& it, uint8_t* smem) {
  using C = ChunkF32<D>;
  constexpr int DC = D / 64;  // groups of four columns a thread
  const int tid = threadIdx.x, tr = tid >> 4, tc = tid & 15;
  float* sq = reinterpret_cast<float*>(smem + C::OFF_Q);
  float* sk = reinterpret_cast<float*>(smem + C::OFF_K);
  float* sv = reinterpret_cast<float*>(smem + C::OFF_V);
  float* sp = reinterpret_cast<float*>(smem + C::OFF_P);
  long long* s_at = reinterpret_cast<long long*>(smem + C::OFF_AT);
  const ChunkSeq s = it.s;
  const int h = it.hg / p.hb, b = it.b;
  // row r of the CTA: tile r / 64, and its token and head in the tile
  auto row_of = [&](int r, int& tok, int& hq) {
    const int rr = r & 63, t = rr / p.gb;
    return chunk_row(p, it.hg, it.t0, it.tokens, r >> 6, t, rr - t * p.gb, tok, hq);
  };
  auto places = [&](int sub) {  // of the slots of 64 from sub * 64 on
    if (tid < C::TS) {
      const int slot = sub * C::TS + tid;
      long long at = -1;
      if (slot < s.held) {
        const int page = page_of(p.c, b, slot / p.c.page_size);
        if (page >= 0) at = page_offset(p.c, page, h) + static_cast<long long>(slot % p.c.page_size) * D;
      }
      s_at[(sub & 1) * C::TS + tid] = at;
    }
  };
  auto fetch = [&](const void* pool, float* to, int stride, int sub, bool any) {
    if (any)
      for (int i = tid; i < C::TS * D / 4; i += 256) {
        const int r = i / (D / 4), c = i % (D / 4) * 4;
        const long long at = s_at[(sub & 1) * C::TS + r];
        cp_async16(smem_u32(to + r * stride + c), static_cast<const float*>(pool) + (at < 0 ? 0 : at + c), at < 0 ? 0 : 16);
      }
    cp_async_commit();
  };
  const int sub0 = it.jb * (kChunkBlock / C::TS), sub1 = it.je * (kChunkBlock / C::TS);
  __syncthreads();  // the item before is through with shared memory
  places(sub0);
  for (int i = tid; i < 16 * MR * D / 4; i += 256) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    int tok, hq;
    float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row_of(r, tok, hq))
      q = *reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + (s.first + tok) * p.q_stride + static_cast<long long>(hq) * D + c);
    *reinterpret_cast<float4*>(sq + r * C::KS + c) = q;
  }
  __syncthreads();
  fetch(p.c.k, sk, C::KS, sub0, true);
  fetch(p.c.v, sv, D, sub0, true);
  int lim[MR];
  float m[MR], l[MR];
  uint64_t o[MR][2 * DC];
  int first_lim = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < MR; ++i) {
    int tok, hq;
    const bool valid = row_of(tr + 16 * i, tok, hq);
    lim[i] = valid ? min(max(s.base + tok + 1, 0), s.held) : 0;
    if (valid) first_lim = min(first_lim, lim[i]);
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < 2 * DC; ++c) o[i][c] = f2(0.f, 0.f);
  }
#pragma unroll 1
  for (int sub = sub0; sub < sub1; ++sub) {
    const bool more = sub + 1 < sub1;
    if (more) places(sub + 1);
    cp_async_wait<1>();
    __syncthreads();
    // ---- scores: even and odd columns summed apart
    uint64_t acc[MR][4];
#pragma unroll
    for (int i = 0; i < MR; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = f2(0.f, 0.f);
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      ulonglong2 k[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) k[e] = *reinterpret_cast<const ulonglong2*>(sk + (tc + 16 * e) * C::KS + d);
#pragma unroll
      for (int i = 0; i < MR; ++i) {
        const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(sq + (tr + 16 * i) * C::KS + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = fma_f2(q.y, k[e].y, fma_f2(q.x, k[e].x, acc[i][e]));
      }
    }
    bool there[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) there[e] = s_at[(sub & 1) * C::TS + tc + 16 * e] >= 0;
    __syncthreads();
    fetch(p.c.k, sk, C::KS, sub + 1, more);
    // ---- softmax
#pragma unroll
    for (int i = 0; i < MR; ++i) {
      float x[4], mx = -INFINITY, sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float a, c;
        f2_split(acc[i][e], a, c);
        x[e] = there[e] && sub * C::TS + tc + 16 * e < lim[i] ? (a + c) * p.scale_log2 : -INFINITY;
        mx = fmaxf(mx, x[e]);
      }
#pragma unroll
      for (int d = 8; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.f : mn, f = ex2(m[i] - base);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = ex2(x[e] - base);
        sum += x[e];
        sp[(tr + 16 * i) * C::PS + tc + 16 * e] = x[e];
      }
#pragma unroll
      for (int d = 8; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      l[i] = fmaf(l[i], f, sum);
      m[i] = mn;
      if (f != 1.f) {
        const uint64_t ff = f2(f, f);
#pragma unroll
        for (int c = 0; c < 2 * DC; ++c) o[i][c] = mul_f2(o[i][c], ff);
      }
    }
    cp_async_wait<1>();
    __syncthreads();
    // ---- O += P V; slots that a row does not see are left out of its sum, where V may hold anything
    const bool cut = (sub + 1) * C::TS > first_lim;
#pragma unroll 2
    for (int j = 0; j < C::TS; j += 4) {
      ulonglong2 v[4][DC];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int c = 0; c < DC; ++c) v[e][c] = *reinterpret_cast<const ulonglong2*>(sv + (j + e) * D + c * 64 + tc * 4);
#pragma unroll
      for (int i = 0; i < MR; ++i) {
        const float4 pr = *reinterpret_cast<const float4*>(sp + (tr + 16 * i) * C::PS + j);
        const float pv[4] = {pr.x, pr.y, pr.z, pr.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (cut && sub * C::TS + j + e >= lim[i]) continue;
          const uint64_t pp = f2(pv[e], pv[e]);
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            o[i][2 * c] = fma_f2(pp, v[e][c].x, o[i][2 * c]);
            o[i][2 * c + 1] = fma_f2(pp, v[e][c].y, o[i][2 * c + 1]);
          }
        }
      }
    }
    __syncthreads();
    fetch(p.c.v, sv, D, sub + 1, more);
  }
  cp_async_wait<0>();
  const bool part = !it.whole();
#pragma unroll
  for (int i = 0; i < MR; ++i) {
    const int r = tr + 16 * i;
    int tok, hq;
    if (!row_of(r, tok, hq)) continue;
    const long long row = s.first + tok;
    if (part) {
      const long long slot = (2ll * blockIdx.x + (it.jb > 0 ? 0 : 1)) * 2 + (r >> 6);
      if (tc == 0) {
        p.part_ml[slot * 128 + (r & 63)] = make_float2(m[i], l[i]);
        if (!it.pair(p)) p.part_ml[(slot + 1) * 128 + (r & 63)] = make_float2(-INFINITY, 0.f);
      }
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        float4 v;
        f2_split(o[i][2 * c], v.x, v.y);
        f2_split(o[i][2 * c + 1], v.z, v.w);
        p.part[slot * (D / 4) * 128 + (c * 16 + tc) * 128 + (r & 63)] = v;
      }
    } else {
      const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
      float* out = static_cast<float*>(p.out) + row * p.out_stride + static_cast<long long>(hq) * D;
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        float4 v;
        f2_split(o[i][2 * c], v.x, v.y);
        f2_split(o[i][2 * c + 1], v.z, v.w);
        v = l[i] == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        *reinterpret_cast<float4*>(out + c * 64 + tc * 4) = v;
      }
      if (tc == 0 && p.lse) p.lse[row * p.Hq + hq] = (m[i] + lg2(l[i])) * 0.6931471805599453f;
    }
  }
}

template <int D>
__global__ void __launch_bounds__(256, 1) chunk_f32_kernel(const __grid_constant__ ChunkParams p) {
  using C = ChunkF32<D>;
  extern __shared__ __align__(128) uint8_t s_ring[];
  grid_wait();
  grid_go();
  ChunkWalk& walk = *reinterpret_cast<ChunkWalk*>(s_ring + C::OFF_WALK + warp_id() * static_cast<int>(sizeof(ChunkWalk)));
  int flags = 0, span_b = 0, span_hg = 0, span_u = 0;
  if (chunk_deal<256>(p, walk)) {
    walk.ahead(p);
    while (walk.next()) {
      const ChunkItem& it = walk.item();
      // rows that the unit's tokens take up, the second tile's behind 64
      const int rows = it.pair(p) ? 64 + (it.tokens - p.tt) * p.gb : it.tokens * p.gb;
      if (rows <= 16) chunk_f32_item<D, 1>(p, it, s_ring);
      else if (rows <= 64) chunk_f32_item<D, 4>(p, it, s_ring);
      else chunk_f32_item<D, 8>(p, it, s_ring);
      if (!it.whole()) {
        const bool begins = it.jb == 0;
        flags |= begins ? SPAN_BEGINS : SPAN_GOES_ON | (it.je == it.nb1 ? SPAN_ENDS : 0);
        if (begins) {
          span_b = it.b;
          span_hg = it.hg;
          span_u = it.u;
        }
      }
      walk.ahead(p);
    }
  }
  if (threadIdx.x == 0) p.span[blockIdx.x] = make_int4(flags, span_b, span_hg, span_u);
}

template <int D, typename T>
static cudaError_t chunk_tc(const ChunkParams& p, cudaStream_t st) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  cudaError_t e = allow_smem<chunk_tc_kernel<D, BF16>>(ChunkCfg<D>::SMEM);
  if (e == cudaSuccess) e = launch_early(chunk_tc_kernel<D, BF16>, dim3(kChunkGrid), kChunkThreads, ChunkCfg<D>::SMEM, st, p);
  if (e == cudaSuccess) e = launch_early(chunk_join_kernel<D, T>, dim3(kChunkGrid, 2 * D / 32), 128, 0, st, p);
  return e;
}

// A 3-D map over 16-bit elements; the first dimension is contiguous, strides in elements.
static cudaError_t chunk_tmap(CUtensorMap* m, const void* base, bool bf16, const long long (&dims)[3],
                              const long long (&strides)[2], int box1, int box2) {
  EncodeTiledFn fn = get_encode_fn();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t d[3] = {static_cast<cuuint64_t>(dims[0]), static_cast<cuuint64_t>(dims[1]),
                           static_cast<cuuint64_t>(dims[2])};
  const cuuint64_t s[2] = {static_cast<cuuint64_t>(strides[0] * 2), static_cast<cuuint64_t>(strides[1] * 2)};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box1), static_cast<cuuint32_t>(box2)}, one[3] = {1, 1, 1};
  const CUresult r = fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                        const_cast<void*>(base), d, s, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// Layout of the workspace.
struct ChunkWs {
  size_t ml, span, bytes;
};
static ChunkWs chunk_ws(const tkb_kv_cache& c) {
  ChunkWs w;
  const size_t tiles = 2 * kChunkGrid * 2;
  w.ml = tiles * 128 * c.D * 4;
  w.span = w.ml + tiles * 128 * sizeof(float2);
  w.bytes = w.span + kChunkGrid * sizeof(int4);
  return w;
}

template <int D>
static cudaError_t chunk_f32(const ChunkParams& p, cudaStream_t st) {
  cudaError_t e = allow_smem<chunk_f32_kernel<D>>(ChunkF32<D>::SMEM);
  if (e == cudaSuccess) e = launch_early(chunk_f32_kernel<D>, dim3(kChunkGrid), 256, ChunkF32<D>::SMEM, st, p);
  if (e == cudaSuccess) e = launch_early(chunk_join_kernel<D, float>, dim3(kChunkGrid, 2 * D / 32), 128, 0, st, p);
  return e;
}

// Two launches.
template <typename T>
static cudaError_t paged_chunk_t(ChunkParams& p, void* workspace, cudaStream_t st) {
  constexpr int tile = sizeof(T) == 4 ? 64 : 128;  // packed rows of a tile
  const int D = p.c.D;
  const ChunkWs w = chunk_ws(p.c);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.part = reinterpret_cast<float4*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + w.ml);
  p.span = reinterpret_cast<int4*>(ws + w.span);
  p.hb = (p.G + tile - 1) / tile;
  p.gb = (p.G + p.hb - 1) / p.hb;
  p.tt = tile / p.gb;
  p.cost = sizeof(T) == 4 ? kCost32 : kCost16;
  if constexpr (sizeof(T) == 4) {
    return D == 64 ? chunk_f32<64>(p, st) : chunk_f32<128>(p, st);
  } else {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    p.gran = kChunkBlock;
    while (p.c.page_size % p.gran) p.gran /= 2;
    cudaError_t e = chunk_tmap(&p.tmQ, p.q, BF16, {D, p.Hq, p.rows}, {D, p.q_stride}, p.gb, p.tt);
    const long long heads = static_cast<long long>(p.c.Hkv) * p.c.page_size;
    if (e == cudaSuccess) e = chunk_tmap(&p.tmK, p.c.k, BF16, {D, heads, p.c.n_pages}, {D, p.c.page_stride}, p.gran, 1);
    if (e == cudaSuccess) e = chunk_tmap(&p.tmV, p.c.v, BF16, {D, heads, p.c.n_pages}, {D, p.c.page_stride}, p.gran, 1);
    if (e != cudaSuccess) return e;
    return D == 64 ? chunk_tc<64, T>(p, st) : chunk_tc<128, T>(p, st);
  }
}

}  // namespace tkb
