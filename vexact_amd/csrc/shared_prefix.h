// Decode attention for groups of sequences that share the pages of a prefix (several answers to one prompt).
//   out = softmax(scale q K^T) V of one query token per sequence over its own keys, of which the first prefix_len[g]
//   lie in pages that all sequences of group g hold.
// The arithmetic is that of attn_core.h, per chunk of 256 keys at absolute positions from a fresh state, chunk states
// folded in ascending order, so the bits are those of the decode kernels on the same block tables. What changes is who
// computes a chunk state: for the whole chunks of a shared prefix the query rows of a group (its sequences times the
// query heads of a kv head) fill the matrix core's 16 columns together, and the chunk's keys are read once per row block
// instead of once per sequence. The chunk at a prefix's end is each sequence's own.
//
// Launch 1: chunk states ("images") of the shared prefixes and, in the same grid behind them, of the sequences' own
// chunks, so that tails of any length fill the chip while the last prefix chunks run. Launch 2: folds a sequence's
// images in ascending order. With enough query rows in the batch a row block instead walks the chunks of its prefix one
// after the other and folds them in registers, which leaves one image instead of one per chunk (attn_shared_walk_kernel).
#pragma once
#include "attn_core.h"

namespace vx {

struct SharedParams {
  const int* group_off;   // [num_groups + 1]: group g = sequences group_off[g] .. group_off[g + 1] - 1
  const int* prefix_len;  // [num_groups]: keys whose pages the group's sequences share
  int num_groups;
  int max_chunks;         // chunks of a prefix that are shared at most
  // images: fp32 accumulators [ceil(dv / 4)][rows] float4, then (m, l) [rows] float2. Shared ones hold a 16-row tile of a
  // group, [tile][kv head][max_chunks]; own ones the G heads of a sequence, [sequence][kv head][max_own].
  float* shared_part;
  int64_t shared_floats;
  float* own_part;
  int64_t own_floats;
  int max_own;
  int blocks;             // launch 1: row blocks per (chunk, kv head), workgroups of the shared part,
  int walked;              // != 0: one folded image per tile of a prefix instead of one per chunk
  int shared_wgs, splits;  // and workgroups that share the own chunks of one (sequence, kv head)
};

static inline int64_t shared_image_floats(int64_t rows, int64_t dv) { return (rows * ((dv + 3) / 4 * 4 + 2) + 3) / 4 * 4; }

struct SharedGroup {
  int seq0, n;  // first sequence, how many
  int tile0;    // first 16-row tile of the group in the workspace
  int chunks;   // whole chunks of keys that are computed once for the group
  int src;      // a sequence of the group that holds all of them: its block table is read
};
// All 64 lanes call it. The shared keys end where the longest sequence of the group ends, whatever prefix_len says, so
// that the block table that is read covers them.
__device__ __forceinline__ SharedGroup shared_group(const AttnParams& p, const SharedParams& s, int g) {
  const int lane = threadIdx.x & 63;
  SharedGroup r;
  r.seq0 = min(max(s.group_off[g], 0), p.num_seqs);
  r.n = min(max(s.group_off[g + 1], r.seq0), p.num_seqs) - r.seq0;
  r.tile0 = (int)((int64_t)r.seq0 * (p.Hq / p.Hkv) / 16) + g;
  int longest = 0;
  r.src = r.seq0;
  for (int b = 0; b < r.n; b += 64) {
    const int len = b + lane < r.n ? min(p.seqused_k[r.seq0 + b + lane], p.max_kv) : 0;
    int m = len;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, __shfl_xor(m, o, 64));
    if (m > longest) {
      longest = m;
      r.src = r.seq0 + b + __builtin_ctzll(__ballot(len == m));
    }
  }
  // a group of one shares nothing: its keys are read once either way
  r.chunks = r.n < 2 ? 0 : min(min(max(s.prefix_len[g], 0), longest) / ATT_CHUNK, s.max_chunks);
  return r;
}
// The group of a sequence, with no chunks if it is in none: the last group that starts at or before it. All 64 lanes.
__device__ __forceinline__ SharedGroup shared_group_of(const AttnParams& p, const SharedParams& s, int seq) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b = 0; b < s.num_groups; b += 64) n += __popcll(__ballot(b + lane < s.num_groups && s.group_off[min(b + lane, s.num_groups - 1)] <= seq));
  SharedGroup r = {};
  if (n > 0) r = shared_group(p, s, n - 1);
  if (seq >= r.seq0 + r.n) r.chunks = 0;
  return r;
}
// Which group row block `item` (rb rows) belongs to, and its place there; -1 behind the last one. The blocks that the
// groups really have are numbered first: the launch has room for a partly filled block per group, and with the unused
// ones in between (every other one where each group fills exactly one) the dispatcher's fixed round of the shader
// engines left half of the CUs without work (16 groups of 16: 138 against 91 us). All 64 lanes call it.
__device__ __forceinline__ int shared_block(const AttnParams& p, const SharedParams& s, int item, int rb, int& place) {
  const int lane = threadIdx.x & 63, G = p.Hq / p.Hkv;
  int base = 0;  // blocks of the groups before this round's
  for (int b = 0; b < s.num_groups; b += 64) {
    int n = 0;
    if (b + lane < s.num_groups) {
      const int s0 = min(max(s.group_off[b + lane], 0), p.num_seqs);
      n = min(max(s.group_off[b + lane + 1], s0), p.num_seqs) - s0;
    }
    const int mine = n < 2 ? 0 : (int)(((int64_t)n * G + rb - 1) / rb);
    int end = mine;  // inclusive sum over the lanes
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(end, o, 64);
      if (lane >= o) end += v;
    }
    const uint64_t after = __ballot(base + end > item);
    if (after) {
      const int l = __builtin_ctzll(after);
      place = item - base - __shfl(end - mine, l, 64);
      return b + l;
    }
    base += __shfl(end, 63, 64);
  }
  return -1;
}

// Launch 1, shared part: workgroup -> (chunk, kv head, row block). Consecutive workgroups go round the eight XCDs, each with
// an L2 of its own: chunk c goes to XCD c % 8, where all row blocks of a (chunk, kv head) follow each other, so the second
// row block of a large group finds the chunk's keys in the L2.
__device__ __forceinline__ void shared_place(int blocks, int Hkv, int& block, int& kvh, int& chunk) {
  const int local = blockIdx.x >> 3;
  block = local % blocks;
  kvh = local / blocks % Hkv;
  chunk = local / blocks / Hkv * 8 + (blockIdx.x & 7);
}
static inline int64_t shared_wgs(int64_t blocks, int Hkv, int chunks) { return blocks * Hkv * ((chunks + 7) / 8 * 8); }

// the state of one 16-row tile in the registers of AttnWave -> an image of `rows` rows (lane r16 = row `row`)
template <class W>
__device__ __forceinline__ void shared_store(const W& w, int t, float* image, int rows, int row, int dv) {
  const int g = (threadIdx.x & 63) >> 4;
  const int d4n = (dv + 3) >> 2;
  float4* ip = (float4*)image + row;
#pragma unroll
  for (int ds = 0; ds < W::NDV; ds++)
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int d4 = 32 * ds + 8 * g + 2 * r + h;
        if (d4 < d4n)
          ip[(int64_t)d4 * rows] = make_float4(w.acc[t][ds * 8 + 4 * h + 0][r], w.acc[t][ds * 8 + 4 * h + 1][r],
                                               w.acc[t][ds * 8 + 4 * h + 2][r], w.acc[t][ds * 8 + 4 * h + 3][r]);
      }
  if (g == 0) ((float2*)(image + (int64_t)4 * d4n * rows))[row] = make_float2(w.m[t], w.l[t]);
}

// Launch 1, own part, workgroups behind the shared ones: wavefront i of WAVES in workgroup (u, z) takes the own chunks
// z WAVES + i, + splits WAVES, ... of pair u = (sequence, kv head). A run of pairs goes to one XCD, so that the keys of the
// partly shared chunk at a prefix's end come from its L2 for all but the first sequence of a group.
template <class ET, int DK, int DV, int QT, int KIND, int WAVES, bool PAD>
__device__ __forceinline__ void attn_own_chunks(const AttnParams& p, const SharedParams& sp) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r16 = lane & 15;
  const int o = blockIdx.x - sp.shared_wgs;  // shared_wgs is a multiple of 8
  const int per = ((int64_t)p.num_seqs * p.Hkv + 7) / 8;  // pairs of an XCD
  const int local = o >> 3, u = (o & 7) * per + local / sp.splits, z = local % sp.splits;
  if (local / sp.splits >= per || u >= p.num_seqs * p.Hkv) return;
  const int seq = u / p.Hkv, kvh = u % p.Hkv, G = p.Hq / p.Hkv;
  const int q0 = p.cu_q[seq], qlen = p.cu_q[seq + 1] - q0;
  const int kv_len = min(p.seqused_k[seq], p.max_kv);
  if (qlen <= 0 || kv_len <= 0) return;
  const int nch = (kv_len + ATT_CHUNK - 1) / ATT_CHUNK;
  const int mine = z * WAVES + wave;  // wave-uniform
  if (mine >= nch) return;            // whatever is shared
  const int first = shared_group_of(p, sp, seq).chunks;
  if (first + mine >= nch) return;
  AttnWave<ET, DK, DV, QT, PAD> w;
  w.init_sizes(p);
  const int64_t tok = q0 + qlen - 1;
#pragma unroll
  for (int t = 0; t < QT; t++) {
    const int hl = 16 * t + r16;
    const bool ok = hl < G;
    w.qpos[t] = ok ? kv_len - 1 : -1;
    w.load_q(t, p.q + tok * p.sqt + (int64_t)(kvh * G + (ok ? hl : 0)) * p.sqh, ok);
  }
  const KVSource<KIND> src = make_source<KIND>(p, seq, kvh, 0, kv_len);
  for (int c = first + mine; c < nch; c += sp.splits * WAVES) {
    w.run_chunk(src, c * ATT_CHUNK, min(c * ATT_CHUNK + ATT_CHUNK, kv_len), kv_len, p.qk_scale);
    float* image = sp.own_part + ((int64_t)u * sp.max_own + (c - first)) * sp.own_floats;
#pragma unroll
    for (int t = 0; t < QT; t++)
      if (16 * t + r16 < G) shared_store(w, t, image, G, 16 * t + r16, w.dv);
  }
}

// Launch 1 for any head size: one wavefront per workgroup; a 16-row tile of a group and chunk, or an own chunk.
template <class ET, int DK, int DV, int QT, int KIND, bool PAD>
__global__ __launch_bounds__(64) void attn_shared_chunks_kernel(AttnParams p, SharedParams sp) {
  if ((int)blockIdx.x >= sp.shared_wgs) {
    attn_own_chunks<ET, DK, DV, QT, KIND, 1, PAD>(p, sp);
    return;
  }
  int block, kvh, chunk, place;
  shared_place(sp.blocks, p.Hkv, block, kvh, chunk);
  const int G = p.Hq / p.Hkv;
  const int gi = shared_block(p, sp, block, 16, place);
  if (gi < 0) return;
  const SharedGroup sg = shared_group(p, sp, gi);
  const int row0 = place * 16;
  if (chunk >= sg.chunks || row0 >= sg.n * G) return;
  const int r16 = threadIdx.x & 15;

  AttnWave<ET, DK, DV, 1, PAD> w;
  w.init_sizes(p);
  const int row = min(row0 + r16, sg.n * G - 1);
  const int seq = sg.seq0 + row / G, head = kvh * G + row % G;
  const int q0 = p.cu_q[seq], qlen = p.cu_q[seq + 1] - q0;
  const bool ok = row0 + r16 < sg.n * G && qlen > 0;
  w.qpos[0] = ok ? min(p.seqused_k[seq], p.max_kv) - 1 : -1;
  w.load_q(0, p.q + (int64_t)(ok ? q0 + qlen - 1 : 0) * p.sqt + (int64_t)head * p.sqh, ok);
  const int keys = sg.chunks * ATT_CHUNK;  // every one of them exists
  const KVSource<KIND> src = make_source<KIND>(p, sg.src, kvh, 0, keys);
  w.run_chunk(src, chunk * ATT_CHUNK, (chunk + 1) * ATT_CHUNK, keys, p.qk_scale);
  if (ok) shared_store(w, 0, sp.shared_part + (((int64_t)(sg.tile0 + place) * p.Hkv + kvh) * sp.max_chunks + chunk) * sp.shared_floats, 16, r16, w.dv);
}

constexpr int SPL_STAGE = 2 * ATT_BLOCK * 256;  // a block's keys and values in LDS
// Direct-to-LDS loads of 64-key blocks by 4 wavefronts: wavefront v brings in keys [16 v, 16 v + 16) of a block, K and V, 4 keys
// (1 KB) per instruction, 8 instructions. Every key exists.
template <int KIND>
struct SharedLoader {
  KVSource<KIND> src;
  uint32_t lds0, koff[4], voff[4];
  int wave, pg_cache, pg_base;  // SRC_FAST: page ids of this wavefront's tile for 64 blocks from pg_base, one per lane

  __device__ __forceinline__ void init(const AttnParams& p, int seq, int kvh, int keys, const uint8_t* lds, int wave_) {
    src = make_source<KIND>(p, seq, kvh, 0, keys);
    wave = wave_;
    const int lane = threadIdx.x & 63;
    lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds + wave * 16 * 256;
    pg_cache = 0;
    pg_base = -64;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int in = 4 * j + (lane >> 4);  // row inside the tile
      koff[j] = (uint32_t)in * (uint32_t)(2 * src.skp) + 16u * (uint32_t)((lane & 15) ^ in);
      voff[j] = (uint32_t)in * (uint32_t)(2 * src.svp) + 16u * (uint32_t)((lane & 15) ^ ((in & 7) << 1));
    }
  }
  static __device__ __forceinline__ const void* uniform(const bf16_t* q) {
    const uint64_t v = (uint64_t)(uintptr_t)q;
    return (const void*)(uintptr_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                                    (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
  }
  __device__ __forceinline__ void issue(int b, int stage) {  // block b of the prefix
    const int key0 = b * ATT_BLOCK + 16 * wave;
    const uint32_t dst = lds0 + stage * SPL_STAGE;
    if constexpr (KIND == SRC_FAST) {
      if (b - pg_base >= 64 || b < pg_base) {  // wave-uniform
        pg_base = b;
        pg_cache = src.bt[min(key0 + (int)(threadIdx.x & 63) * ATT_BLOCK, src.last) >> src.shift];
      }
      const int pg = __builtin_amdgcn_readlane(pg_cache, b - pg_base), off = key0 & (src.ps - 1);
      const void* kt = uniform(src.kbase + (int64_t)pg * src.skb + (int64_t)off * src.skp);
      const void* vt = uniform(src.vbase + (int64_t)pg * src.svb + (int64_t)off * src.svp);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        lds_load16_sv(dst + 4 * j * 256, koff[j], kt);
        lds_load16_sv(dst + 4 * j * 256 + ATT_BLOCK * 256, voff[j], vt);
      }
    } else {
      const typename KVSource<KIND>::Tiles tl = {};
      const int lane = threadIdx.x & 63;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int in = 4 * j + (lane >> 4);
        lds_load16_v(dst + 4 * j * 256, src.krow(tl, key0, 0, in) + 8 * ((lane & 15) ^ in));
        lds_load16_v(dst + 4 * j * 256 + ATT_BLOCK * 256, src.vrow(tl, key0, 0, in) + 8 * ((lane & 15) ^ ((in & 7) << 1)));
      }
    }
  }
};

// Query rows lr0 .. lr0 + 16 TILES - 1 of a group and kv head as MFMA operands, with their last visible keys (-1: no such
// row) and the smallest of them per tile (blocks that end at or before it need no mask).
template <int TILES>
__device__ __forceinline__ void shared_load_queries(const AttnParams& p, const SharedGroup& sg, int kvh, int lr0, int keys,
                                                    uint4 (&qf)[TILES][4], int (&qpos)[TILES], int (&qpos_min)[TILES]) {
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const int G = p.Hq / p.Hkv, rows = sg.n * G;
#pragma unroll
  for (int t = 0; t < TILES; t++) {
    const int lr = lr0 + 16 * t + r16;
    const int row = min(lr, rows - 1);
    const int seq = sg.seq0 + row / G, head = kvh * G + row % G;
    const int q0 = p.cu_q[seq], qlen = p.cu_q[seq + 1] - q0;
    const bool ok = lr < rows && qlen > 0;
    qpos[t] = ok ? min(p.seqused_k[seq], p.max_kv) - 1 : -1;
    const bf16_t* qp = p.q + (int64_t)(ok ? q0 + qlen - 1 : 0) * p.sqt + (int64_t)head * p.sqh + 8 * g;
#pragma unroll
    for (int s = 0; s < 4; s++) qf[t][s] = ldg16(qp + 32 * s, ok);
    int v = ok ? qpos[t] : keys;  // rows that do not exist need no mask
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
    qpos_min[t] = __builtin_amdgcn_readfirstlane(v);
  }
}

// One 64-key block from its LDS stage (keys, then values, laid out as attn_prefill_lds_kernel has them): scores, online
// softmax and P V of TILES 16-row tiles.
template <int TILES>
__device__ __forceinline__ void shared_block_compute(const uint8_t* ks, int kb, float scale, const uint4 (&qf)[TILES][4], const int (&qpos)[TILES],
                                                   const int (&qpos_min)[TILES], float (&m)[TILES], float (&l)[TILES], f32x4 (&acc)[TILES][8]) {
  constexpr int KS = 4;
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const uint8_t* vs = ks + ATT_BLOCK * 256;
  f32x4 st[TILES][4];
#pragma unroll
  for (int t = 0; t < TILES; t++)
#pragma unroll
    for (int tt = 0; tt < 4; tt++) st[t][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < KS; s++)
#pragma unroll
    for (int tt = 0; tt < 4; tt++) {
      const uint4 kfr = *(const uint4*)(ks + (16 * tt + r16) * 256 + (((4 * s + g) ^ r16) * 16));
#pragma unroll
      for (int t = 0; t < TILES; t++) st[t][tt] = mfma16(kfr, qf[t][s], st[t][tt]);
    }
  uint4 pf[TILES][2];
#pragma unroll
  for (int t = 0; t < TILES; t++)
    attn_softmax_tile<ElemBF16>(st[t], kb, scale, qpos[t], m[t], l[t], acc[t], pf[t], kb + ATT_BLOCK - 1 <= qpos_min[t]);
#pragma unroll
  for (int ch = 0; ch < 2; ch++)
#pragma unroll
    for (int f = 0; f < 8; f++) {
      const int byte = 32 * f + 8 * (r16 & 3);
      const int row_lo = 32 * ch + 4 * g + (r16 >> 2), row_hi = row_lo + 16;
      const v4s_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) v4s_t*)(vs + row_lo * 256 + (((byte >> 4) ^ ((row_lo & 7) << 1)) * 16) + (byte & 15)));
      const v4s_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) v4s_t*)(vs + row_hi * 256 + (((byte >> 4) ^ ((row_hi & 7) << 1)) * 16) + (byte & 15)));
      const uint2 lo2 = __builtin_bit_cast(uint2, lo), hi2 = __builtin_bit_cast(uint2, hi);
      const uint4 vf = make_uint4(lo2.x, lo2.y, hi2.x, hi2.y);
#pragma unroll
      for (int t = 0; t < TILES; t++) acc[t][f] = mfma16(vf, pf[t][ch], acc[t][f]);
    }
}

// Launch 1 for bf16 heads of 128: the chunk's keys and values are shared by the workgroup through LDS: 4 wavefronts with TILES
// 16-row tiles each, 64-key blocks brought in by direct-to-LDS loads into one of two 32 KB stages (two workgroups on a
// CU cover each other's waits), operands, softmax and P V as in attn_prefill_lds_kernel (same layouts and swizzles, same
// bits). Every wavefront loads the 16 keys of one tile of the block. A chunk is read once per 64 TILES query rows.
template <int TILES, int QT, int KIND>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void attn_shared_chunks_lds_kernel(AttnParams p, SharedParams sp) {
  if ((int)blockIdx.x >= sp.shared_wgs) {
    attn_own_chunks<ElemBF16, 128, 128, QT, KIND, 4, false>(p, sp);
    return;
  }
  constexpr int D = 128, KS = D / 32, RB = 64 * TILES;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * SPL_STAGE];
  int block, kvh, chunk, place;
  shared_place(sp.blocks, p.Hkv, block, kvh, chunk);
  const int G = p.Hq / p.Hkv;
  const int gi = shared_block(p, sp, block, RB, place);
  if (gi < 0) return;
  const SharedGroup sg = shared_group(p, sp, gi);
  const int rows = sg.n * G, row0 = place * RB;
  if (chunk >= sg.chunks || row0 >= rows) return;  // uniform over the block
  constexpr int nb = ATT_CHUNK / ATT_BLOCK;
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int keys = sg.chunks * ATT_CHUNK;  // every one of them exists

  SharedLoader<KIND> ld;
  ld.init(p, sg.src, kvh, keys, lds, wave);
  const int b0 = chunk * nb;
  ld.issue(b0, 0);
  ld.issue(b0 + 1, 1);

  // ---- this wavefront's query tiles
  uint4 qf[TILES][KS];
  int qpos[TILES], qpos_min[TILES];
  shared_load_queries<TILES>(p, sg, kvh, row0 + 16 * wave * TILES, keys, qf, qpos, qpos_min);
  float m[TILES], l[TILES];
  f32x4 acc[TILES][8];
#pragma unroll
  for (int t = 0; t < TILES; t++) {
    m[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const bool any = row0 + 16 * wave * TILES < rows;  // wave-uniform: a wavefront without rows only loads
#pragma unroll
  for (int b = 0; b < nb; b++) {
    // 8 loads per block and wavefront, the youngest of which are those of block b + 1: at most 8 outstanding means that
    // block b has landed
    if (b + 1 < nb) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (any) shared_block_compute<TILES>(lds + (b & 1) * SPL_STAGE, chunk * ATT_CHUNK + b * ATT_BLOCK, p.qk_scale, qf, qpos, qpos_min, m, l, acc);
    __syncthreads();  // everyone has read the stage
    if (b + 2 < nb) ld.issue(b0 + b + 2, b & 1);
  }

  // lane (r16 = query row, g) holds dims 16 f + 4 g .. + 3 of fragment f
#pragma unroll
  for (int t = 0; t < TILES; t++) {
    const int lr = row0 + 16 * (wave * TILES + t);
    if (lr + r16 >= rows) continue;
    float* image = sp.shared_part + (((int64_t)(sg.tile0 + (lr >> 4)) * p.Hkv + kvh) * sp.max_chunks + chunk) * sp.shared_floats;
#pragma unroll
    for (int f = 0; f < 8; f++)
      ((float4*)image)[(4 * f + g) * 16 + r16] = make_float4(acc[t][f][0], acc[t][f][1], acc[t][f][2], acc[t][f][3]);
    if (g == 0) ((float2*)(image + D * 16))[r16] = make_float2(m[t], l[t]);
  }
}

// Launch 1 for bf16 heads of 128 in large batches: a workgroup of 4 wavefronts (64 query rows) walks all shared chunks of its
// group and folds them in registers: one image per tile in place of one per chunk. Four 32 KB stages keep three blocks of
// loads in flight, one barrier per block. The row blocks 2 i and 2 i + 1 of a kv head go to one XCD, so that a group of 128
// rows reads its keys from HBM once.
constexpr int SPW_STAGES = 4;
static inline int64_t walk_wgs(int64_t blocks, int Hkv) { return 16 * (((blocks + 1) / 2 * Hkv + 7) / 8); }
template <int QT, int KIND>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void attn_shared_walk_kernel(AttnParams p, SharedParams sp) {
  if ((int)blockIdx.x >= sp.shared_wgs) {
    attn_own_chunks<ElemBF16, 128, 128, QT, KIND, 4, false>(p, sp);
    return;
  }
  constexpr int D = 128, KS = D / 32, RB = 64;
  extern __shared__ __attribute__((aligned(1024))) uint8_t sw_lds[];
  const int local = blockIdx.x >> 3, v = (local >> 1) * 8 + (blockIdx.x & 7);
  const int block = 2 * (v / p.Hkv) + (local & 1), kvh = v % p.Hkv;
  int place;
  const int gi = shared_block(p, sp, block, RB, place);
  if (gi < 0) return;
  const SharedGroup sg = shared_group(p, sp, gi);
  const int rows = sg.n * (p.Hq / p.Hkv), row0 = place * RB;
  if (sg.chunks == 0 || row0 >= rows) return;  // uniform over the block
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int keys = sg.chunks * ATT_CHUNK, nblk = sg.chunks * (ATT_CHUNK / ATT_BLOCK);
  SharedLoader<KIND> ld;
  ld.init(p, sg.src, kvh, keys, sw_lds, wave);
  uint4 qf[1][KS];
  int qpos[1], qpos_min[1];
  shared_load_queries<1>(p, sg, kvh, row0 + 16 * wave, keys, qf, qpos, qpos_min);
#pragma unroll
  for (int b = 0; b < SPW_STAGES - 1; b++) ld.issue(b, b);  // a chunk has four blocks: they exist
  float M = -INFINITY, L = 0.f;
  f32x4 ACC[8];
#pragma unroll
  for (int i = 0; i < 8; i++) ACC[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int b0 = 0; b0 < nblk; b0 += 4) {
    float m[1] = {-INFINITY}, l[1] = {0.f};
    f32x4 acc[1][8];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[0][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int b = b0 + i;
      // 8 loads per block and wavefront, in order: all but the youngest two blocks' have landed
      if (b + 2 < nblk) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
      else if (b + 1 < nblk) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();  // block b is there for everyone, and everyone is done with block b - 1
      if (b + 3 < nblk) ld.issue(b + 3, (i + 3) & 3);
      shared_block_compute<1>(sw_lds + i * SPL_STAGE, b * ATT_BLOCK, p.qk_scale, qf, qpos, qpos_min, m, l, acc);
    }
    float Mn, A, B;
    fold_scales(M, m[0], Mn, A, B);
    L = fold_add(L, A, l[0], B);
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
      for (int r = 0; r < 4; r++) ACC[i][r] = fold_add(ACC[i][r], A, acc[0][i][r], B);
    M = Mn;
  }
  const int lr = row0 + 16 * wave;
  if (lr + r16 >= rows) return;
  float* image = sp.shared_part + ((int64_t)(sg.tile0 + (lr >> 4)) * p.Hkv + kvh) * sp.shared_floats;
#pragma unroll
  for (int f = 0; f < 8; f++) ((float4*)image)[(4 * f + g) * 16 + r16] = make_float4(ACC[f][0], ACC[f][1], ACC[f][2], ACC[f][3]);
  if (g == 0) ((float2*)(image + D * 16))[r16] = make_float2(M, L);
}

// Launch 2: one workgroup per (sequence, kv head), a thread per (head, 4 dims): shared chunks, then own ones, in ascending
// order with the fold of the decode kernels; a sequence without keys gets zeros.
template <class ET, bool PAD>
__global__ __launch_bounds__(256) void attn_shared_fold_kernel(AttnParams p, SharedParams sp) {
  const int kvh = blockIdx.x, seq = blockIdx.y, G = p.Hq / p.Hkv;
  const int q0 = p.cu_q[seq], qlen = p.cu_q[seq + 1] - q0;
  if (qlen <= 0) return;
  const int kv_len = min(p.seqused_k[seq], p.max_kv);
  const int64_t tok = q0 + qlen - 1;
  const int d4n = (p.dv + 3) >> 2, nelem = G * d4n;
  const SharedGroup sg = shared_group_of(p, sp, seq);
  const int nch = kv_len > 0 ? (kv_len + ATT_CHUNK - 1) / ATT_CHUNK : 0;
  const int first = min(sg.chunks, nch);  // a sequence shorter than its group's prefix ends inside it
  const int ns = sp.walked ? min(first, 1) : first;
  for (int e = threadIdx.x; e < nelem; e += blockDim.x) {
    const int hl = e % G, d4 = e / G;
    float4 A4 = make_float4(0.f, 0.f, 0.f, 0.f);
    float M = -INFINITY, L = 0.f;
    // n images, `stride` floats apart: this thread's four accumulators at `a`, its row's (m, l) at `b`; U in flight
    auto fold = [&](const float* a, const float* b, int n, int64_t stride) {
      constexpr int U = 16;
      for (int c0 = 0; c0 < n; c0 += U) {
        float4 av[U];
        float2 mv[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
          const int64_t o = (c0 + u < n ? c0 + u : c0) * stride;
          av[u] = *(const float4*)(a + o);
          mv[u] = *(const float2*)(b + o);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
          if (c0 + u < n) {
            float Mn, A, B;
            fold_scales(M, mv[u].x, Mn, A, B);
            L = fold_add(L, A, mv[u].y, B);
            A4.x = fold_add(A4.x, A, av[u].x, B);
            A4.y = fold_add(A4.y, A, av[u].y, B);
            A4.z = fold_add(A4.z, A, av[u].z, B);
            A4.w = fold_add(A4.w, A, av[u].w, B);
            M = Mn;
          }
        }
      }
    };
    if (ns > 0) {
      const int row = (seq - sg.seq0) * G + hl;
      const float* image = sp.shared_part + ((int64_t)(sg.tile0 + (row >> 4)) * p.Hkv + kvh) * (sp.walked ? 1 : sp.max_chunks) * sp.shared_floats;
      fold(image + ((int64_t)d4 * 16 + (row & 15)) * 4, image + (int64_t)4 * d4n * 16 + 2 * (row & 15), ns, sp.shared_floats);
    }
    if (nch > first) {
      const float* image = sp.own_part + ((int64_t)seq * p.Hkv + kvh) * sp.max_own * sp.own_floats;
      fold(image + ((int64_t)d4 * G + hl) * 4, image + (int64_t)4 * d4n * G + 2 * hl, nch - first, sp.own_floats);
    }
    uint2 pk = make_uint2(0u, 0u);
    if (nch > 0) {
      pk.x = ET::pack2(A4.x / L, A4.y / L);
      pk.y = ET::pack2(A4.z / L, A4.w / L);
    }
    attn_st4<PAD>(p.o + tok * p.sot + (int64_t)(kvh * G + hl) * p.soh, 4 * d4, pk, p.dv, p.elem);
  }
}

template <class ET, int DK, int DV, int QT, int KIND, bool PAD>
static int launch_shared_prefix_t(const AttnParams& p, SharedParams sp, hipStream_t stream) {
  const int G = p.Hq / p.Hkv;
  const int64_t rows = (int64_t)p.num_seqs * G, pairs = (int64_t)p.num_seqs * p.Hkv;
  constexpr bool LDS = ET::kDtype == 0 && DK == 128 && DV == 128 && !PAD;
  constexpr int WAVES = LDS ? 4 : 1;
  // row tiles per wavefront: one where an average group has at most 64 rows, else two
  const int tiles = LDS && rows > 64 * (int64_t)sp.num_groups ? 2 : 1;
  // Walk the prefixes where that occupies half of the CUs: 64 rows of one kv head per workgroup
  const bool walk = LDS && rows * p.Hkv >= 64 * 128;
  sp.walked = walk;
  sp.blocks = (int)(rows / (16 * WAVES * (walk ? 1 : tiles)) + sp.num_groups);
  const int64_t swgs = sp.num_groups == 0 || sp.max_chunks == 0 ? 0 : walk ? walk_wgs(sp.blocks, p.Hkv) : shared_wgs(sp.blocks, p.Hkv, sp.max_chunks);
  // about 4096 wavefronts for the own chunks, at most one per chunk
  sp.splits = (int)std::max<int64_t>(1, std::min<int64_t>((sp.max_own + WAVES - 1) / WAVES, 4096 / (pairs * WAVES)));
  const int64_t owgs = (pairs + 7) / 8 * 8 * sp.splits;
  if (swgs + owgs > 0x7fffffff) return VX_ERR_UNSUPPORTED;
  sp.shared_wgs = (int)swgs;
  const unsigned grid = (unsigned)(swgs + owgs);
  if constexpr (LDS) {
    if (walk) {
      constexpr int LDSB = SPW_STAGES * SPL_STAGE;
      static DeviceOnce once;
      const int dev = once.slot();
      if (once.need(dev)) {
        if (hipFuncSetAttribute((const void*)attn_shared_walk_kernel<QT, KIND>, hipFuncAttributeMaxDynamicSharedMemorySize, LDSB) != hipSuccess) {
          (void)hipGetLastError();
          return VX_ERR_LAUNCH;
        }
        once.mark(dev);
      }
      attn_shared_walk_kernel<QT, KIND><<<grid, 256, LDSB, stream>>>(p, sp);
    } else if (tiles == 2) attn_shared_chunks_lds_kernel<2, QT, KIND><<<grid, 256, 0, stream>>>(p, sp);
    else attn_shared_chunks_lds_kernel<1, QT, KIND><<<grid, 256, 0, stream>>>(p, sp);
  } else {
    attn_shared_chunks_kernel<ET, DK, DV, QT, KIND, PAD><<<grid, 64, 0, stream>>>(p, sp);
  }
  const int rc = launch_status();
  if (rc != VX_OK) return rc;
  const int nelem = G * ((p.dv + 3) / 4);
  attn_shared_fold_kernel<ET, PAD><<<dim3(p.Hkv, p.num_seqs), nelem > 128 ? 256 : nelem > 64 ? 128 : 64, 0, stream>>>(p, sp);
  return launch_status();
}

template <class ET, int DK, int DV, bool PAD>
static int launch_shared_prefix(const AttnParams& p, const SharedParams& sp, hipStream_t stream) {
  const bool fast = p.page_shift >= 4;  // page size a power of two >= 16
  if (p.Hq / p.Hkv <= 16)
    return fast ? launch_shared_prefix_t<ET, DK, DV, 1, SRC_FAST, PAD>(p, sp, stream) : launch_shared_prefix_t<ET, DK, DV, 1, SRC_GENERIC, PAD>(p, sp, stream);
  return fast ? launch_shared_prefix_t<ET, DK, DV, 2, SRC_FAST, PAD>(p, sp, stream) : launch_shared_prefix_t<ET, DK, DV, 2, SRC_GENERIC, PAD>(p, sp, stream);
}

// in translation units of their own (compile time); DKb / DVb as for launch_attn_bf16_padded
int launch_shared_prefix_bf16_padded(const AttnParams& p, const SharedParams& sp, int DKb, int DVb, hipStream_t stream);
int launch_shared_prefix_f16(const AttnParams& p, const SharedParams& sp, int DKb, int DVb, hipStream_t stream);

}  // namespace vx
