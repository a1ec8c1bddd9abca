// paged_attn.cu — causal attention over the paged Q4_0 KV cache.
//
// Row i of a sequence's n rows sits at position p_i = len - n + i and sees
// positions 0..p_i. With codes q (integers -8..7) and block scales d,
//
//   s_t = scale * sum_w dK[t,w] * (sum_{j in group w} Q_j qK[t,j])
//   O_j = sum_t (p_t dV[t,w(j)]) qV[t,j] / sum_t p_t,   p_t = exp(s_t - max)
//
// The integers are exact in fp16 and bf16, so the tensor cores multiply codes
// and the scales are applied outside in fp32: to the accumulators of each
// 32-dimension group for K, to the probabilities for V. Nothing of the cache is
// rounded a second time.
//
// Decode form: a warp takes 16 tokens at a time. S = Q K^T is mma.m16n8k16 with
// tokens as columns; its accumulators are already the column operand of
// O^T = V^T P^T, so nothing is transposed and O^T of 8 rows is 32 registers.
// Both operands that are not codes are fp16: queries, each row first scaled by a
// power of two so that its largest element is near 2^13, and p 2^F dV with F such
// that 2^F max(dV) is below 2^14 and 2^F at most 2^15 (F follows the largest
// scale met so far, as max does the largest score, and comes off at the end).
// fp32 calls keep both as hi + lo pairs, off by at most 2^-21 of the value, or
// 2^-25 2^-F where that is larger; bf16 queries are exact in one fp16 (down to
// 2^-27 of the row's largest), and p 2^F and its product with dV in one fp16
// each are off by at most 2^-10, a quarter of the bf16 output's own half step, or
// 2^-25 2^-F where that is larger: 2^-38 of the largest dV that the row's tile sees.
//
// Work: the blocks of all (sequence, KV head, row tile) units are laid end to
// end in chunks of 64 tokens and cut into equal runs, one per CTA, so uneven
// lengths cost nothing; a unit cut between CTAs leaves partial (max, sum, O)
// records that a second kernel joins in chunk order, so results do not depend on
// timing.
//
// Measured: one fp32 sequence of 131072 tokens, 64 heads over 8 of 128: 58 us, 2.6
// TB/s of cache; 64 bf16 sequences of 512 to 8192: 72 us, 3.0 TB/s; 16 fp32 sequences
// of up to 4096 with 5 rows and 32 KV heads: 51 us. The main loop alone runs at 3.7
// TB/s: about 400 instructions for a warp's 16 tokens of 128, a third of them the
// widening of codes, at 55 to 60 % of the issue slots. The rest is waiting: 16 warps per
// SM, each in a chain of products, two shuffles, votes, exponentials and products again.
// Before it come 4.6 us until the first block is there, after it 4 to 6 us for the join.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged.cuh"

namespace mlb {

namespace {

constexpr int kDecWarps = 4;
constexpr int kDecThreads = kDecWarps * 32;
constexpr int kChunkTokens = kPagedBlock * kDecWarps;  // one block per warp
constexpr int kStages = 5;                    // blocks on their way per warp, and in use
// A unit counts for this many chunks more than it has: its queries, the join of its
// warps and its result take a CTA about as long as three (64 uneven sequences: 1: 80 us,
// 2: 76, 3: 73, 5: 73).
constexpr int kUnitSlots = 3;
constexpr int kMaxSegs = 32;                  // segments of a run listed at a time

// CTAs per SM: 128 registers a thread for one 8-row tile, 168 for two.
__host__ __device__ constexpr int dec_ctas(int nt) { return nt > 1 ? 3 : 4; }

// Part of a CTA's run: chunks [chunk0, chunk1) of one (sequence, KV head, row tile).
struct Seg {
  int seq, head, tile, chunk0, chunk1, chunks, len, n, row0, record;
  long long pos0;
};

// a / b of non-negative numbers; 32-bit division where that will do (a quarter of the
// instructions, and every warp does a few per segment).
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
__device__ __forceinline__ long long run_begin(long long total, int i, int n) {
  return quotient(total * i, n);
}

// F of the largest V scale met so far: 2^F d < 2^14, and 2^F itself within fp16.
__device__ __forceinline__ int shift_of(uint32_t d_bits) {
  return min(28 - max((int)(d_bits >> 10), 1), 15);
}
// NT 8-row tiles per unit. SPLIT: queries and P dV as hi + lo pairs.
template <int G, int NT, class T>
__global__ void __launch_bounds__(kDecThreads, dec_ctas(NT))
    paged_attn_decode_kernel(PagedAttnArgs a) {
  constexpr bool SPLIT = sizeof(T) == 4;
  constexpr int R = 8 * NT;
  constexpr int MT = SPLIT ? NT : (NT + 1) / 2;
  constexpr int BLOCK = 576 * G;
  constexpr int D = 32 * G;
  constexpr int REC = R * D + 2 * R;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint4 queries[MT * G * 2 * 32];  // MMA A words of the tile, by (m-tile, w, k half, lane)
  __shared__ long long warp_sums[kDecWarps];
  __shared__ long long found_base;
  __shared__ int found_seq;
  __shared__ int slot_ok[kDecWarps][kStages];
  __shared__ Seg segs[kMaxSegs];

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int cta = blockIdx.x;

  // total work, this CTA's run, and the sequence that holds its begin (one look at
  // the sequences where a block has a thread for each)
  const bool few = a.seqs.n_seqs <= kDecThreads;
  long long total = 0, cost = 0, incl = 0;
  for (int s0 = 0; s0 < a.seqs.n_seqs; s0 += kDecThreads) {
    const int s = s0 + threadIdx.x;
    cost = s < a.seqs.n_seqs ? seq_work(a, s, R, kChunkTokens, kUnitSlots).cost : 0;
    total += cost;
  }
  incl = block_scan<kDecThreads>(total, warp_sums);
  if (threadIdx.x == kDecThreads - 1) found_base = incl;
  __syncthreads();
  total = found_base;
  __syncthreads();
  const int nrun = (int)min((long long)gridDim.x, total);
  int4* split = a.split + 2 * cta;
  if (cta >= nrun) {
    if (threadIdx.x == 0 && !a.whole) split[0] = make_int4(0, 0, 0, 0);
    return;
  }
  const long long begin = run_begin(total, cta, nrun), end = run_begin(total, cta + 1, nrun);
  const long long prev = cta > 0 ? run_begin(total, cta - 1, nrun) : 0;
  if (few) {
    if (cost > 0 && begin >= incl - cost && begin < incl) {
      found_seq = threadIdx.x;
      found_base = incl - cost;
    }
    __syncthreads();
  } else {
    long long base = 0;
    for (int s0 = 0; s0 < a.seqs.n_seqs; s0 += kDecThreads) {
      const int s = s0 + threadIdx.x;
      cost = s < a.seqs.n_seqs ? seq_work(a, s, R, kChunkTokens, kUnitSlots).cost : 0;
      incl = block_scan<kDecThreads>(cost, warp_sums) + base;
      if (cost > 0 && begin >= incl - cost && begin < incl) {
        found_seq = s;
        found_base = incl - cost;
      }
      if (threadIdx.x == kDecThreads - 1) warp_sums[0] = incl;
      __syncthreads();
      base = warp_sums[0];
      __syncthreads();
      if (base > begin) break;
    }
  }
  int seq = found_seq;
  long long base = found_base;
  SeqWork sw = seq_work(a, seq, R, kChunkTokens, kUnitSlots);
  if (threadIdx.x == 0 && !a.whole) split[0] = make_int4(0, 0, 0, 0);

  uint8_t* ring = smem + warp * (kStages * BLOCK);
  const int bpp = a.cache.page_size / kPagedBlock;

  for (long long at = begin; at < end;) {
    // the next segments of the run, every thread in step, thread 0 noting them
    int n_segs = 0;
    while (at < end && n_segs < kMaxSegs) {
      while (at >= base + sw.cost) {  // next sequence with rows
        base += sw.cost;
        ++seq;
        sw = seq_work(a, seq, R, kChunkTokens, kUnitSlots);
      }
      const long long u = quotient(at - base, sw.slots);  // unit within the sequence
      const long long unit_begin = base + u * sw.slots;
      if (at - unit_begin >= sw.chunks) {  // the slots past its chunks stand for its ends
        at = unit_begin + sw.slots;
        continue;
      }
      Seg sg;
      sg.seq = seq;
      sg.head = (int)quotient(u, sw.tiles);
      sg.tile = (int)(u - (long long)sg.head * sw.tiles);
      sg.chunk0 = (int)(at - unit_begin);
      sg.chunk1 = a.whole ? sw.chunks : (int)min((long long)sw.chunks, end - unit_begin);
      sg.chunks = sw.chunks;
      sg.len = sw.len;
      sg.n = sw.n;
      sg.row0 = sw.row0;
      sg.pos0 = sw.pos0;
      sg.record = at == begin ? 0 : 1;
      if (threadIdx.x == 0) {
        segs[n_segs] = sg;
        if (at == begin && unit_begin < begin && prev <= unit_begin) {
          // this CTA holds the second part of a unit that an earlier one began;
          // the last part is with the last run that begins before the unit ends
          const long long unit_end = unit_begin + sw.chunks;
          const int last = (int)quotient(unit_end * nrun + total - 1, total) - 1;
          split[0] = make_int4(last - cta + 2, prev == unit_begin ? 0 : 1, sg.head, sg.tile);
          split[1] = make_int4(sw.row0, sw.n, 0, 0);
        }
      }
      ++n_segs;
      at = unit_begin + (a.whole ? 1 : sg.chunk1);
    }
    if (n_segs == 0) break;
    __syncthreads();

    // copies, running ahead of the arithmetic across segments: block 4 chunk + warp
    int is = 0, ic = segs[0].chunk0, iw = 0, slot_in = 0;
    int at_block = -1;  // place in the layer of this lane's block of the next 32, -1: none
    auto issue = [&]() {
      if (is < n_segs) {
        const Seg& sg = segs[is];
        if (iw == 0) {
          const int bl = (ic + lane) * kDecWarps + warp;
          at_block = -1;
          if (bl * kPagedBlock < sg.len) {
            const int p = bl / bpp;
            const int page = a.seqs.table[(size_t)sg.seq * a.seqs.max_pages + p];
            if (page >= 0 && page < a.cache.n_pages)
              at_block = (page * a.cache.kv + sg.head) * bpp + (bl - p * bpp);
          }
        }
        const int from = __shfl_sync(0xffffffffu, at_block, iw);
        if (lane == 0) slot_ok[warp][slot_in] = from >= 0;
        if (from >= 0) {
          const uint8_t* src = a.cache.layer + (size_t)from * BLOCK + lane * 16;
          uint8_t* dst = ring + slot_in * BLOCK + lane * 16;
#pragma unroll
          for (int i = 0; i < BLOCK / 512; ++i) cp_async16(dst + i * 512, src + i * 512);
          if (BLOCK % 512 != 0 && lane < BLOCK % 512 / 16)
            cp_async16(dst + BLOCK / 512 * 512, src + BLOCK / 512 * 512);
        }
        slot_in = slot_in + 1 == kStages ? 0 : slot_in + 1;
        iw = (iw + 1) & 31;
        if (++ic == sg.chunk1) {
          ++is;
          iw = 0;
          if (is < n_segs) ic = segs[is].chunk0;
        }
      }
      cp_async_commit();
    };
    int slot = 0;

    for (int si = 0; si < n_segs; ++si) {
      const Seg& sg = segs[si];

      // queries: row r of the tile is flat row tile R + r = token * group + head
      float rs[NT];  // score factor of this lane's row in each 8-row tile
      int vis[NT];   // positions it sees
      int vis_min = 0x7fffffff, vis_max = 0;  // of the tile's rows (rows past the last: none)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const long long flat = (long long)sg.tile * R + t * 8 + g;
        const bool live = flat < (long long)sg.n * a.group;
        const int i = live ? (int)quotient(flat, a.group) : 0;
        const int hq = sg.head * a.group + (live ? (int)(flat - (long long)i * a.group) : 0);
        vis[t] = live ? seen_by(sg.pos0, i, sg.len) : 0;
        if (live) vis_min = min(vis_min, vis[t]);
        vis_max = max(vis_max, vis[t]);
        const T* row = live ? static_cast<const T*>(a.q) + (long long)(sg.row0 + i) * a.q_stride +
                                  (size_t)hq * a.cache.head_dim
                            : nullptr;
        float e[G][8];
        if (si == 0 && t == 0) {
          // the first queries are asked for before the copies that would be ahead of
          // them in the memory's queue
          load_query_elements<G, T>(row, a.cache.head_dim, c, e);
#pragma unroll
          for (int i = 0; i < kStages - 1; ++i) issue();
        } else {
          load_query_elements<G, T>(row, a.cache.head_dim, c, e);
        }
        const int sh = query_shift<G>(e);
        rs[t] = pow2(-sh) * a.scale_log2;
        // the warps share the tile; each makes and writes its part of the words
        const float sf = pow2(sh);
#pragma unroll
        for (int w = 0; w < G; ++w)
          if (w % kDecWarps == warp) {
            uint32_t hi[4], lo[4];
            query_words(e[w], sf, SPLIT, hi, lo);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              uint4& q = queries[(((SPLIT ? t : t / 2) * G + w) * 2 + k) * 32 + lane];
              if (SPLIT) {
                q = make_uint4(hi[2 * k], lo[2 * k], hi[2 * k + 1], lo[2 * k + 1]);
              } else if (t & 1) {
                q.y = hi[2 * k];
                q.w = hi[2 * k + 1];
              } else {
                q = make_uint4(hi[2 * k], 0u, hi[2 * k + 1], 0u);
              }
            }
          }
      }
      vis_min = __reduce_min_sync(0xffffffffu, vis_min);
      vis_max = __reduce_max_sync(0xffffffffu, vis_max);
      __syncthreads();

      float o[NT][2 * G][4];
      float m[NT];
      float2 l[NT];
      uint32_t dtop = 0;           // largest V scale so far, fp16 bits
      int shift = shift_of(dtop);  // F: O is in units of 2^-F
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        m[t] = -INFINITY;
        l[t] = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < 2 * G; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[t][i][j] = 0.0f;
      }

      // One block of 16 tokens. WHOLE: every row of the tile sees all of them.
      auto step = [&](auto whole_c, const uint8_t* block, int tok0) {
        constexpr bool WHOLE = decltype(whole_c)::value;

        // scores: s[t][n-tile] = tokens 8 nt + 2 c, + 1
        float2 s[NT][2];
        {
          uint32_t kw[2][G], ks[2][G];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            lds_words<G>(block + (nt * 8 + g) * 16 * G + c * 4 * G, kw[nt]);
            lds_words<G>(block + 512 * G + (nt * 4 + c) * 4 * G, ks[nt]);
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = make_float2(0.f, 0.f);
#pragma unroll
          for (int w = 0; w < G; ++w) {
            uint32_t b[2][4];
            codes_f16(kw[0][w], b[0]);
            codes_f16(kw[1][w], b[1]);
            const float2 d0 = __half22float2(u32_as_h2(ks[0][w]));
            const float2 d1 = __half22float2(u32_as_h2(ks[1][w]));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              const uint4 u0 = queries[((mt * G + w) * 2 + 0) * 32 + lane];
              const uint4 u1 = queries[((mt * G + w) * 2 + 1) * 32 + lane];
              const uint32_t q0[4] = {u0.x, u0.y, u0.z, u0.w}, q1[4] = {u1.x, u1.y, u1.z, u1.w};
              float acc[2][4];
#pragma unroll
              for (int nt = 0; nt < 2; ++nt) {
                mma_16816_z(acc[nt], q0, b[nt][0], b[nt][1]);
                mma_16816(acc[nt], q1, b[nt][2], b[nt][3]);
              }
#pragma unroll
              for (int nt = 0; nt < 2; ++nt) {
                const float2 d = nt ? d1 : d0;
                const float2 x = make_float2(acc[nt][0], acc[nt][1]);
                const float2 y = make_float2(acc[nt][2], acc[nt][3]);
                if (SPLIT) {
                  s[mt][nt] = fma2(d, add2(x, y), s[mt][nt]);
                } else {
                  constexpr int LAST = NT - 1;
                  const int t1 = 2 * mt + 1 < NT ? 2 * mt + 1 : LAST;
                  s[2 * mt][nt] = fma2(d, x, s[2 * mt][nt]);
                  if (2 * mt + 1 < NT) s[t1][nt] = fma2(d, y, s[t1][nt]);
                }
              }
            }
          }
        }

        // online softmax; hidden[t] bit 2 nt + parity: token not seen by the row
        uint32_t hidden[NT], hidden_all = 0xfu;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          hidden[t] = 0;
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            s[t][nt] = mul2(s[t][nt], make_float2(rs[t], rs[t]));
            if (!WHOLE) {
              const int tok = tok0 + nt * 8 + 2 * c;
              if (tok >= vis[t]) {
                s[t][nt].x = -INFINITY;
                hidden[t] |= 1u << (2 * nt);
              }
              if (tok + 1 >= vis[t]) {
                s[t][nt].y = -INFINITY;
                hidden[t] |= 2u << (2 * nt);
              }
            }
          }
          hidden_all &= hidden[t];
          float mx = fmaxf(fmaxf(s[t][0].x, s[t][0].y), fmaxf(s[t][1].x, s[t][1].y));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          if (__any_sync(0xffffffffu, mx > m[t])) {
            const float mn = fmaxf(m[t], mx);
            const float al = m[t] == -INFINITY ? 0.0f : ex2(m[t] - mn);
            m[t] = mn;
            l[t].x *= al;
            l[t].y *= al;
            const float a0 = __shfl_sync(0xffffffffu, al, 8 * c);      // row 2 c
            const float a1 = __shfl_sync(0xffffffffu, al, 8 * c + 4);  // row 2 c + 1
#pragma unroll
            for (int i = 0; i < 2 * G; ++i) {
              o[t][i][0] *= a0;
              o[t][i][1] *= a1;
              o[t][i][2] *= a0;
              o[t][i][3] *= a1;
            }
          }
          const float ref = m[t] == -INFINITY ? 0.0f : -m[t];  // -inf: nothing seen yet
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            s[t][nt] = add2(s[t][nt], make_float2(ref, ref));
            s[t][nt].x = ex2(s[t][nt].x);
            s[t][nt].y = ex2(s[t][nt].y);
            l[t] = add2(l[t], s[t][nt]);
          }
        }

        // V scales; F follows the largest that some row sees
        uint32_t vd[2][G];
        __half2 dmax = u32_as_h2(0u);
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          lds_words<G>(block + 544 * G + (nt * 4 + c) * 4 * G, vd[nt]);
          const uint32_t keep = WHOLE ? 0xffffffffu
                                      : (hidden_all >> (2 * nt) & 1 ? 0u : 0xffffu) |
                                            (hidden_all >> (2 * nt) & 2 ? 0u : 0xffff0000u);
#pragma unroll
          for (int w = 0; w < G; ++w) dmax = __hmax2(dmax, u32_as_h2(vd[nt][w] & keep));
        }
        const uint32_t db = h2_as_u32(dmax);
        const uint32_t dnow = __reduce_max_sync(0xffffffffu, max(db & 0xffffu, db >> 16));
        if (dnow > dtop) {
          dtop = dnow;
          const int now = shift_of(dtop);
          if (now != shift) {
            const float f = pow2(now - shift);
            shift = now;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int i = 0; i < 2 * G; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[t][i][j] *= f;
          }
        }

        // p 2^F as fp16 pairs (and what they leave)
        const float up = pow2(shift);
        uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const float2 x = mul2(s[t][nt], make_float2(up, up));
            ph[t][nt] = pack_f16(x.x, x.y);
            if (SPLIT) {
              const float2 h = __half22float2(u32_as_h2(ph[t][nt]));
              pl[t][nt] = pack_f16(x.x - h.x, x.y - h.y);
            }
          }

        // O^T += V^T (P dV)^T
        uint32_t v0[G], v1[G];
        lds_words<G>(block + 256 * G + lane * 4 * G, v0);
        lds_words<G>(block + 384 * G + lane * 4 * G, v1);
#pragma unroll
        for (int w = 0; w < G; ++w) {
          uint32_t x0[4], x1[4];
          codes_f16(v0[w], x0);
          codes_f16(v1[w], x1);
          const uint32_t a0[4] = {x0[0], x0[1], x1[0], x1[1]};
          const uint32_t a1[4] = {x0[2], x0[3], x1[2], x1[3]};
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // P dV = hi + lo: hi d rounded, its remainder exact, lo d on top
              const __half2 d = u32_as_h2(vd[j][w]), h = u32_as_h2(ph[t][j]);
              const __half2 x = __hmul2(h, d);
              hi[j] = h2_as_u32(x);
              if (SPLIT)
                lo[j] = h2_as_u32(__hfma2(u32_as_h2(pl[t][j]), d, __hfma2(h, d, __hneg2(x))));
              if (!WHOLE) {  // a hidden token's scale may be anything
                const uint32_t hb = hidden[t] >> (2 * j);
                const uint32_t keep = (hb & 1 ? 0u : 0xffffu) | (hb & 2 ? 0u : 0xffff0000u);
                hi[j] &= keep;
                if (SPLIT) lo[j] &= keep;
              }
            }
            mma_16816(o[t][2 * w], a0, hi[0], hi[1]);
            mma_16816(o[t][2 * w + 1], a1, hi[0], hi[1]);
            if (SPLIT) {
              mma_16816(o[t][2 * w], a0, lo[0], lo[1]);
              mma_16816(o[t][2 * w + 1], a1, lo[0], lo[1]);
            }
          }
        }
      };

      // every chunk but the last leaves its slot to the copies at once; the last
      // one's slot takes the warp's result first
      const int chunk1 = sg.chunk1;
      for (int chunk = sg.chunk0;;) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncwarp();
        const int tok0 = (chunk * kDecWarps + warp) * kPagedBlock;
        if (slot_ok[warp][slot] && tok0 < vis_max) {
          if (tok0 + kPagedBlock <= vis_min)
            step(std::true_type{}, ring + slot * BLOCK, tok0);
          else
            step(std::false_type{}, ring + slot * BLOCK, tok0);
        }
        __syncwarp();
        if (++chunk == chunk1) break;
        issue();
        slot = slot + 1 == kStages ? 0 : slot + 1;
      }

      // join the warps, 8 rows by D / 2 dimensions at a time: each leaves (O, max,
      // sum) of its tokens in the slot that it has just used
      const float down = pow2(-shift);
      const bool complete = sg.chunk0 == 0 && chunk1 == sg.chunks;
      float* part = a.partial + ((size_t)cta * 2 + sg.record) * REC;
      constexpr int H = D / 2;
      auto record_of = [&](int w) {
        return reinterpret_cast<float*>(smem + (w * kStages + slot) * BLOCK);
      };
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float sum = l[t].x + l[t].y;
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        float* rec = record_of(warp);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (c == 0) {
            rec[8 * H + g] = m[t];
            rec[8 * H + 8 + g] = sum;
          }
          // lane holds rows 2 c, 2 c + 1 of every m-tile: two dimensions each
#pragma unroll
          for (int i = 0; i < G; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              *reinterpret_cast<float2*>(rec + (2 * c + e) * H + 16 * i + 2 * g) =
                  make_float2(o[t][h * G + i][e] * down, o[t][h * G + i][2 + e] * down);
          __syncthreads();
          for (int i = threadIdx.x; i < 8 * (H / 2); i += kDecThreads) {
            const int r = i / (H / 2), x0 = (i - r * (H / 2)) * 2;
            // pair x0 of m-tile x0 / 16: dims 32 w + 4 g + 2 (m-tile & 1)
            const int mt = h * G + x0 / 16, d0 = 32 * (mt >> 1) + 2 * (x0 % 16) + 2 * (mt & 1);
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < kDecWarps; ++w) mx = fmaxf(mx, record_of(w)[8 * H + r]);
            float all = 0.0f;
            float2 x = make_float2(0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kDecWarps; ++w) {
              const float mw = record_of(w)[8 * H + r];
              const float f = mw == mx ? 1.0f : ex2(mw - mx);
              const float2 y = *reinterpret_cast<const float2*>(record_of(w) + r * H + x0);
              all = fmaf(f, record_of(w)[8 * H + 8 + r], all);
              x.x = fmaf(f, y.x, x.x);
              x.y = fmaf(f, y.y, x.y);
            }
            if (complete) {
              const long long flat = (long long)sg.tile * R + t * 8 + r;
              if (flat < (long long)sg.n * a.group && d0 < a.cache.head_dim) {
                const int tk = (int)quotient(flat, a.group);
                const int hq = sg.head * a.group + (int)(flat - (long long)tk * a.group);
                const float f = all == 0.0f ? 0.0f : 1.0f / all;  // sees nothing: zeros
                store_act2(static_cast<T*>(a.out) + (long long)(sg.row0 + tk) * a.out_stride +
                               (size_t)hq * a.cache.head_dim + d0,
                           x.x * f, x.y * f);
              }
            } else {
              *reinterpret_cast<float2*>(part + (t * 8 + r) * D + d0) = x;
              if (d0 == 0) {
                part[R * D + t * 8 + r] = mx;
                part[R * D + R + t * 8 + r] = all;
              }
            }
          }
          __syncthreads();
        }
      }
      issue();
      slot = slot + 1 == kStages ? 0 : slot + 1;
    }
    cp_async_wait_all();
    __syncthreads();  // segs and the slots are used again
  }
  pdl_launch_dependents();
}

// Joins the parts of units that were cut between CTAs: block (i, y) joins row y
// of the unit whose second part CTA i holds. The warps take every fourth part,
// so that up to 24 of them are on their way at a time; the order is fixed.
template <int G, int NT, class T>
__global__ void __launch_bounds__(kDecThreads, 8) paged_attn_join_kernel(PagedAttnArgs a) {
  constexpr int R = 8 * NT;
  constexpr int D = 32 * G;
  constexpr int REC = R * D + 2 * R;
  __shared__ float xs[kDecWarps][D], sums[kDecWarps], tops[kDecWarps];
  pdl_wait();
  const int4 s0 = a.split[2 * blockIdx.x], s1 = a.split[2 * blockIdx.x + 1];
  const int parts = s0.x, head = s0.z, tile = s0.w, row0 = s1.x, n = s1.y;
  if (parts == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = blockIdx.y;
  const long long flat = (long long)tile * R + r;
  if (flat >= (long long)n * a.group) return;
  const float* first = a.partial + ((size_t)(blockIdx.x - 1) * 2 + s0.y) * REC;
  const float* rest = a.partial + (size_t)blockIdx.x * 2 * REC;  // part p >= 1: + 2 (p - 1) REC
  auto rec = [&](int p) { return p == 0 ? first : rest + (size_t)(p - 1) * 2 * REC; };
  // this warp's parts, six at a time (eight cost the registers of resident CTAs), each
  // batch under the largest maximum so far
  float mx = -INFINITY, sum = 0.0f, x[G];
#pragma unroll
  for (int w = 0; w < G; ++w) x[w] = 0.0f;
  for (int p0 = warp; p0 < parts; p0 += 6 * kDecWarps) {
    float m[6], l[6], y[6][G];
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      const int p = p0 + i * kDecWarps;
      const float* q = rec(min(p, parts - 1));
      m[i] = p < parts ? q[R * D + r] : -INFINITY;
      l[i] = p < parts ? q[R * D + R + r] : 0.0f;
#pragma unroll
      for (int w = 0; w < G; ++w) y[i][w] = q[r * D + 32 * w + lane];
    }
    float top = mx;
#pragma unroll
    for (int i = 0; i < 6; ++i) top = fmaxf(top, m[i]);
    const float f0 = mx == top ? 1.0f : ex2(mx - top);
    mx = top;
    sum *= f0;
#pragma unroll
    for (int w = 0; w < G; ++w) x[w] *= f0;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      if (p0 + i * kDecWarps >= parts) continue;
      const float f = m[i] == mx ? 1.0f : ex2(m[i] - mx);
      sum = fmaf(f, l[i], sum);
#pragma unroll
      for (int w = 0; w < G; ++w) x[w] = fmaf(f, y[i][w], x[w]);
    }
  }
#pragma unroll
  for (int w = 0; w < G; ++w) xs[warp][32 * w + lane] = x[w];
  if (lane == 0) {
    sums[warp] = sum;
    tops[warp] = mx;
  }
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= a.cache.head_dim) return;
  sum = 0.0f;
  mx = -INFINITY;
  float y = 0.0f;
#pragma unroll
  for (int w = 0; w < kDecWarps; ++w) mx = fmaxf(mx, tops[w]);
#pragma unroll
  for (int w = 0; w < kDecWarps; ++w) {
    const float f = tops[w] == mx ? 1.0f : ex2(tops[w] - mx);
    sum = fmaf(f, sums[w], sum);
    y = fmaf(f, xs[w][d], y);
  }
  y *= sum == 0.0f ? 0.0f : 1.0f / sum;
  const int tk = (int)(flat / a.group);
  const int hq = head * a.group + (int)(flat - (long long)tk * a.group);
  T* out = static_cast<T*>(a.out) + (long long)(row0 + tk) * a.out_stride +
           (size_t)hq * a.cache.head_dim;
  if constexpr (sizeof(T) == 4)
    out[d] = y;
  else
    out[d] = __float2bfloat16_rn(y);
}

// 8-row tiles per unit: two where the call's rows per KV head and sequence are
// more than 8 on average, so that each block's codes are widened once for 16.
int dec_tiles(int n_rows, int n_seqs, int group) {
  return (long long)n_rows * group > 8LL * n_seqs ? 2 : 1;
}

int dec_grid(int sms, int nt) { return sms * dec_ctas(nt); }

// Whether a call takes the prompt form. Both forms' times grow with the length, so
// what decides is the time per 64 tokens, from the average rows per sequence and KV
// head: the decode form spreads row tiles of 16 over 3 CTAs per SM, 1.5 us each
// (fp32: 2.05), the prompt form runs waves of one CTA per SM, 1.65 us for up to 256
// rows (fp32: 2.1 for 128). Measured, decode / prompt us, bf16: 16 sequences of 4096
// with 8 KV heads, 32 rows 72 / 90, 128 rows 225 / 86; one sequence of 4096, 512 rows
// 72 / 93, 1024 rows 124 / 94; of 32768, 1024 rows 744 / 638. All at head_dim 128.
// Averages do not see a long sequence with a row beside a prompt: the prompt form cuts
// no tile's length, so such a call is as long as its longest sequence (bf16, 32 heads
// over 8: 512 rows of a prompt and one row over 131072 tokens 2645 us, as two calls
// 25 + 54; 2048 rows and 63 rows over 512 to 7952 tokens 479, as two 67 + 93).
bool prompt_form(int act, int n_rows, int n_seqs, int kv, int group, int sms) {
  const bool f32 = act == MLB_ACT_F32;
  const long long units = (long long)n_seqs * kv;
  const long long rows = ((long long)n_rows * group + n_seqs - 1) / n_seqs;
  const long long per_cta = f32 ? 128 : 256;
  const double decode = (double)(units * ((rows + 15) / 16)) * (f32 ? 2.05 : 1.5) / (3 * sms);
  const long long ctas = units * ((rows + per_cta - 1) / per_cta);
  const double prompt = (double)((ctas + sms - 1) / sms) * (f32 ? 2.1 : 1.65);
  return prompt < decode;
}

// Whether units stay whole, so that the second kernel and the workspace fall away:
// where the page table holds 256 tokens, or 512 and there are 64 units. A CTA takes
// about 13 us per 1000 tokens of a unit. Measured, whole / cut us, fp32, 32 heads over 8
// KV heads, one row each: 1 sequence of 128 tokens 7.4 / 9.5, of 256 9.3 / 9.5, of 500
// 12.6 / 9.6; 8 sequences of 500 13.1 / 13.5, of 1000 19.9 / 13.8; 64 of 500 21.0 / 26.6.
// All at head_dim 128.
bool whole_units(int max_pages, int page_size, int n_seqs, int kv) {
  const long long tokens = (long long)max_pages * page_size;
  return tokens <= 256 || (tokens <= 512 && (long long)n_seqs * kv >= 64);
}

size_t dec_workspace(int grid, int groups, int nt) {
  const size_t rec = (size_t)8 * nt * 32 * groups + 16 * nt;
  return (size_t)grid * (2 * sizeof(int4) + 2 * rec * sizeof(float));
}

template <int G, int NT, class T>
void launch_decode(const PagedAttnArgs& a, int grid, int device_id, cudaStream_t stream) {
  constexpr size_t smem = (size_t)kDecWarps * kStages * 576 * G;
  static_assert((8 * 16 * G + 16) * 4 <= 576 * G, "a record of 8 rows and half the dimensions fits a slot");
  allow_smem(paged_attn_decode_kernel<G, NT, T>, smem, device_id);
  paged_attn_decode_kernel<G, NT, T><<<grid, kDecThreads, smem, stream>>>(a);
  MLB_CUDA(cudaGetLastError());
  if (a.whole) return;
  launch_pdl(paged_attn_join_kernel<G, NT, T>, dim3(grid, 8 * NT), dim3(kDecThreads), 0, stream,
             true, a);
}

template <class T>
void decode_dispatch(const PagedAttnArgs& a, int groups, int nt, int grid, int device_id,
                     cudaStream_t s) {
  switch (groups * 4 + nt) {
    case 4 + 1: return launch_decode<1, 1, T>(a, grid, device_id, s);
    case 4 + 2: return launch_decode<1, 2, T>(a, grid, device_id, s);
    case 8 + 1: return launch_decode<2, 1, T>(a, grid, device_id, s);
    case 8 + 2: return launch_decode<2, 2, T>(a, grid, device_id, s);
    case 12 + 1: return launch_decode<3, 1, T>(a, grid, device_id, s);
    case 12 + 2: return launch_decode<3, 2, T>(a, grid, device_id, s);
    case 16 + 1: return launch_decode<4, 1, T>(a, grid, device_id, s);
    default: return launch_decode<4, 2, T>(a, grid, device_id, s);
  }
}

void check_heads(const char* who, int n_heads, int kv) {
  if (n_heads <= 0) invalid(std::string(who) + ": n_heads must be positive");
  if (n_heads % kv != 0) invalid(std::string(who) + ": n_heads must be divisible by n_kv_heads");
}

}  // namespace

}  // namespace mlb

using namespace mlb;

extern "C" int mlb_paged_attention_workspace(int act_type, int n_rows, int n_seqs, int n_heads,
                                             int n_kv_heads, int head_dim, int page_size,
                                             int max_pages, int device_id, size_t* bytes) {
  return guarded([&] {
    const char* who = "CudaPagedAttention";
    if (!bytes) invalid("CudaPagedAttention: null output");
    paged_check_act(who, act_type);
    paged_check_shape(who, page_size, n_kv_heads, head_dim);
    check_heads(who, n_heads, n_kv_heads);
    if (n_rows < 0 || n_seqs < 0) invalid("CudaPagedAttention: negative row or sequence count");
    if (max_pages <= 0) invalid("CudaPagedAttention: page_table must have at least one column");
    DeviceScope scope(device_id);
    const int group = n_heads / n_kv_heads, sms = sm_count(device_id);
    const int nt = dec_tiles(n_rows, n_seqs, group);
    *bytes = n_rows == 0 || n_seqs == 0 || whole_units(max_pages, page_size, n_seqs, n_kv_heads) ||
                     prompt_form(act_type, n_rows, n_seqs, n_kv_heads, group, sms)
                 ? 0
                 : dec_workspace(dec_grid(sms, nt), paged_groups(head_dim), nt);
  });
}

extern "C" int mlb_paged_attention(const void* pages, int n_layers, int n_pages, int page_size,
                                   int n_kv_heads, int head_dim, int layer, int act_type,
                                   const void* q, long long q_stride, int n_heads, int n_rows,
                                   int n_seqs, const int* row_offsets, const int* seq_lens,
                                   const int* page_table, int max_pages, float scale, void* out,
                                   long long out_stride, void* workspace, size_t workspace_bytes,
                                   int device_id, void* stream) {
  return guarded([&] {
    const char* who = "CudaPagedAttention";
    PagedAttnArgs a;
    a.cache = paged_cache(who, const_cast<void*>(pages), n_layers, n_pages, page_size, n_kv_heads,
                          head_dim, layer);
    a.seqs = paged_seqs(who, n_rows, n_seqs, row_offsets, seq_lens, page_table, max_pages,
                        page_size);
    paged_check_act(who, act_type);
    check_heads(who, n_heads, n_kv_heads);
    const float scale_log2 = scale * 1.4426950408889634f;
    if (!std::isfinite(scale_log2)) invalid("CudaPagedAttention: scale must be finite");
    if (n_rows > 0) {
      paged_check_rows(who, "q", q, q_stride, n_heads, head_dim, act_type);
      paged_check_rows(who, "out", out, out_stride, n_heads, head_dim, act_type);
      const long long row = (long long)n_heads * head_dim;
      if (rows_overlap(q, q_stride, row, out, out_stride, row, n_rows, act_type))
        invalid("CudaPagedAttention: q and out must not overlap");
    }
    DeviceScope scope(device_id);
    if (n_rows == 0 || n_seqs == 0) return;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.n_heads = n_heads;
    a.group = n_heads / n_kv_heads;
    a.scale_log2 = scale_log2;
    a.whole = false;
    a.split = nullptr;
    a.partial = nullptr;
    a.wait_cycles = 0;
    a.never = 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int sms = sm_count(device_id);
    if (prompt_form(act_type, n_rows, n_seqs, n_kv_heads, a.group, sms)) {
      paged_prompt_launch(a, act_type, device_id, s);
      return;
    }
    const int groups = paged_groups(head_dim);
    const int nt = dec_tiles(n_rows, n_seqs, a.group);
    const int most = dec_grid(sms, nt);
    a.whole = whole_units(max_pages, page_size, n_seqs, n_kv_heads);
    if (!a.whole) {
      if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
          workspace_bytes < dec_workspace(most, groups, nt))
        invalid("CudaPagedAttention: workspace is null, unaligned or too small");
      a.split = static_cast<int4*>(workspace);
      a.partial = reinterpret_cast<float*>(a.split + 2 * (size_t)most);
    }
    // no more CTAs than units or chunks that the page table and the rows can make
    const long long tiles =
        ((long long)n_rows * a.group + 8 * nt - 1) / (8 * nt) + n_seqs;
    const long long chunks =
        a.whole ? 1 : ((long long)max_pages * page_size + kChunkTokens - 1) / kChunkTokens;
    const int grid = (int)std::min<long long>(most, tiles * n_kv_heads * chunks);
    if (act_type == MLB_ACT_BF16)
      decode_dispatch<__nv_bfloat16>(a, groups, nt, grid, device_id, s);
    else
      decode_dispatch<float>(a, groups, nt, grid, device_id, s);
  });
}
