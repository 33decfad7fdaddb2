// Decode attention for groups of sequences that share the pages of a prefix (several answers to one prompt).
//   out = softmax(scale q K^T) V of one query token per sequence over its own keys, of which the first prefix_len[g]
//   lie in pages that all sequences of group g hold.
// The arithmetic is that of attn_core.h, per chunk of 256 keys at absolute positions from a fresh state, chunk states
// folded in ascending order, so the bits are those of the decode kernels on the same block tables. What changes is who
// computes a chunk state: for the whole chunks of a shared prefix the query rows of a group (its sequences times the
// query heads of a kv head) fill the matrix core's 16 columns together, and the chunk's keys are read once per row block
// instead of once per sequence. The chunk at a prefix's end is each sequence's own, and so is the chunk in which a sequence
// shorter than its group's prefix ends: every row that a shared chunk is computed for, and later read for, sees all of its
// keys, so nothing is masked there, and keys behind a sequence's end may hold anything.
//
// Launch 1: chunk states ("images") of the shared prefixes and, in the same grid behind them, of the sequences' own
// chunks, so that tails of any length fill the chip while the last prefix chunks run. Launch 2: folds a sequence's
// images in ascending order. (A row block that walks its chunks one after the other and folds them in registers needs no
// images of them, but its steps are a chain, and at 16 groups of 16 it leaves half of the CUs without one: level at 8192
// query rows, 4 times slower for one group of 64 on 32768 keys.)
// At a full decode batch both launches run at the rate of a large copy: what they move is the prefixes once (241 MB at 16
// groups of 16 on prefixes about 7400, 32 / 4 heads), their images twice (2 x 131 MB) and the tails (300 MB): 138 + 33 us.
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
  // launch 1: workgroups of the shared part that have work if the prefixes are equally long, of the own part (multiples of
  // 8), chunks that a shared workgroup takes, workgroups that share the own chunks of one (sequence, kv head)
  int shared_sure, own_first, own_wgs, cpw, splits;
};

static inline int64_t shared_image_floats(int64_t rows, int64_t dv) { return (rows * ((dv + 3) / 4 * 4 + 2) + 3) / 4 * 4; }

struct SharedGroup {
  int seq0, n;  // first sequence, how many
  int tile0;    // first 16-row tile of the group in the workspace
  int chunks;   // whole chunks of keys that are computed once for the group
  int src;      // a sequence of the group, with a query token, that holds all of them: its block table is read
};
// The offsets and prefix lengths of 64 groups from `b` on, one per lane, so that whichever is wanted needs no second round
// trip to memory.
struct SharedLane {
  int seq0, n, prefix;
};
__device__ __forceinline__ SharedLane shared_lane(const AttnParams& p, const SharedParams& s, int b) {
  const int g = b + (threadIdx.x & 63);
  SharedLane l = {p.num_seqs, 0, 0};
  if (g < s.num_groups) {
    const int o0 = s.group_off[g], o1 = s.group_off[g + 1];
    l.prefix = s.prefix_len[g];
    l.seq0 = min(max(o0, 0), p.num_seqs);
    l.n = min(max(o1, l.seq0), p.num_seqs) - l.seq0;
  }
  return l;
}
// The group in lane `from` of l (group g). All 64 lanes call it. The shared keys end where the longest sequence of the
// group ends, whatever prefix_len says, so that the block table that is read covers them. A slot without a query token
// counts as empty: its length and block table may be those of a sequence that has ended, its pages another's by now.
__device__ __forceinline__ SharedGroup shared_group(const AttnParams& p, const SharedParams& s, const SharedLane& l, int from, int g) {
  const int lane = threadIdx.x & 63;
  SharedGroup r;
  r.seq0 = __builtin_amdgcn_readlane(l.seq0, from);
  r.n = __builtin_amdgcn_readlane(l.n, from);
  r.tile0 = (int)((int64_t)r.seq0 * (p.Hq / p.Hkv) / 16) + g;
  int longest = 0;
  r.src = r.seq0;
  for (int b = 0; b < r.n; b += 64) {
    int len = 0;
    if (b + lane < r.n) {
      const int i = r.seq0 + b + lane, used = min(p.seqused_k[i], p.max_kv);
      len = p.cu_q[i + 1] > p.cu_q[i] ? used : 0;
    }
    int m = len;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, __shfl_xor(m, o, 64));
    if (m > longest) {
      longest = m;
      r.src = r.seq0 + b + __builtin_ctzll(__ballot(len == m));
    }
  }
  // a group of one shares nothing: its keys are read once either way
  r.chunks = r.n < 2 ? 0 : min(min(max(__builtin_amdgcn_readlane(l.prefix, from), 0), longest) / ATT_CHUNK, s.max_chunks);
  return r;
}
// The group of a sequence, with no chunks if it is in none: the last group that starts at or before it. All 64 lanes.
__device__ __forceinline__ SharedGroup shared_group_of(const AttnParams& p, const SharedParams& s, int seq) {
  SharedLane l, hit = {};
  int from = -1, g = 0;
  for (int b = 0; b < s.num_groups; b += 64) {
    l = shared_lane(p, s, b);
    const int left = s.num_groups - b;
    const uint64_t at = __ballot(l.seq0 <= seq) & (left < 64 ? (1ull << left) - 1 : ~0ull);
    if (!at) break;
    hit = l;
    from = 63 - __builtin_clzll(at);
    g = b + from;
  }
  SharedGroup r = {};
  if (from >= 0) r = shared_group(p, s, hit, from, g);
  if (seq >= r.seq0 + r.n) r.chunks = 0;
  return r;
}
// Shared workgroup `index` -> its kv head, first chunk and row block (rb rows): the group and the block's place in it; false
// if there is nothing for it. All 64 lanes call it. An XCD has an L2 of its own: chunk c belongs to XCD c % 8, where all row
// blocks of a (chunk, kv head) follow each other, so the second row block of a large group finds the chunk's keys in the
// L2. A workgroup takes cpw chunks, 8 apart. Only the blocks that the groups really have are numbered, so the workgroups
// that the launch has too many (a partly filled block per group: its host knows no sizes) come last. Between the others
// they cost a workgroup's slot for three trips to memory, and where every other one is empty (16 groups that fill a block
// each) the dispatcher's fixed round of the shader engines leaves half of the CUs without work (138 against 91 us).
__device__ __forceinline__ bool shared_unit(const AttnParams& p, const SharedParams& s, int index, int rb, SharedGroup& sg, int& place, int& kvh, int& chunk) {
  const int lane = threadIdx.x & 63, G = p.Hq / p.Hkv;
  SharedLane gl;
  int mine, end;  // blocks of this lane's group; of this and the lower lanes' groups
  auto read = [&](int b) {
    gl = shared_lane(p, s, b);
    end = mine = gl.n < 2 ? 0 : (int)(((int64_t)gl.n * G + rb - 1) / rb);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(end, o, 64);
      if (lane >= o) end += v;
    }
    return __builtin_amdgcn_readlane(end, 63);
  };
  int total = 0;
  for (int b = 0; b < s.num_groups; b += 64) total += read(b);
  if (total == 0) return false;
  const int local = index >> 3, pair = local / total;
  kvh = pair % p.Hkv;
  chunk = pair / p.Hkv * (8 * s.cpw) + (index & 7);
  if (chunk >= s.max_chunks) return false;
  int item = local - pair * total;
  for (int b = 0;; b += 64) {
    const int here = s.num_groups <= 64 ? total : read(b);
    if (item < here) {
      const int l = __builtin_ctzll(__ballot(end > item));
      place = item - __builtin_amdgcn_readlane(end - mine, l);
      sg = shared_group(p, s, gl, l, b + l);
      return true;
    }
    item -= here;
  }
}

// Launch 1 holds shared and own workgroups; returns the index within the kind, -1 - index for an own one. In front are those
// that surely have work, a block or more per group and the first own workgroup of every pair, alternating in proportion, so
// that a CU runs one that waits for the matrix core beside one that waits for memory; behind them the further own
// workgroups, then the rest of the shared ones, most of which have nothing to do (against all of both kinds alternating,
// with every pair's own workgroups together: 16 groups of 16 175 -> 170 us, 128 sequences in 32 groups 87 -> 68, 45 in 7
// uneven groups 35 -> 32). Always eight consecutive ids, which go round the eight XCDs, are of one kind.
__device__ __forceinline__ int shared_kind(const SharedParams& sp) {
  const int grp = blockIdx.x >> 3, in = blockIdx.x & 7;
  const int64_t first = sp.own_first >> 3, all = first + (sp.shared_sure >> 3), rest = (sp.own_wgs - sp.own_first) >> 3;
  if (grp >= all + rest) return (int)(grp - first - rest) * 8 + in;
  if (grp >= all) return -1 - ((int)(grp - all + first) * 8 + in);
  const int before = (int)(grp * first / all), upto = (int)((grp + 1) * first / all);
  return upto > before ? -1 - (before * 8 + in) : (grp - before) * 8 + in;
}

// workgroups for `blocks` row blocks
static inline int64_t shared_wgs(int64_t blocks, int Hkv, int chunks, int cpw) { return blocks * Hkv * ((chunks + 8 * cpw - 1) / (8 * cpw) * 8); }

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

// Launch 1, own part: wavefront i of WAVES in workgroup (u, z) takes the own chunks
// z WAVES + i, + splits WAVES, ... of pair u = (sequence, kv head); the first workgroups of all pairs come first. A run of pairs goes to one XCD, so that the keys of the
// partly shared chunk at a prefix's end come from its L2 for all but the first sequence of a group.
template <class ET, int DK, int DV, int QT, int KIND, int WAVES, bool PAD>
__device__ __forceinline__ void attn_own_chunks(const AttnParams& p, const SharedParams& sp, int o) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r16 = lane & 15;
  const int per = ((int64_t)p.num_seqs * p.Hkv + 7) / 8;  // pairs of an XCD
  const int local = o >> 3, u = (o & 7) * per + local % per, z = local / per;
  if (u >= p.num_seqs * p.Hkv) return;
  const int seq = u / p.Hkv, kvh = u % p.Hkv, G = p.Hq / p.Hkv;
  const int q0 = p.cu_q[seq], qlen = p.cu_q[seq + 1] - q0;
  const int kv_len = min(p.seqused_k[seq], p.max_kv);
  if (qlen <= 0 || kv_len <= 0) return;
  const int nch = (kv_len + ATT_CHUNK - 1) / ATT_CHUNK;
  const int mine = z * WAVES + wave;  // wave-uniform
  if (mine >= nch) return;            // whatever is shared
  const int first = min(shared_group_of(p, sp, seq).chunks, kv_len / ATT_CHUNK);
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
  const int index = shared_kind(sp);
  if (index < 0) {
    attn_own_chunks<ET, DK, DV, QT, KIND, 1, PAD>(p, sp, -1 - index);
    return;
  }
  int kvh, chunk, place;
  const int G = p.Hq / p.Hkv;
  SharedGroup sg;
  if (!shared_unit(p, sp, index, 16, sg, place, kvh, chunk)) return;
  const int row0 = place * 16;
  if (chunk >= sg.chunks || row0 >= sg.n * G) return;
  const int r16 = threadIdx.x & 15;

  AttnWave<ET, DK, DV, 1, PAD> w;
  w.init_sizes(p);
  const int row = min(row0 + r16, sg.n * G - 1);
  const int seq = sg.seq0 + row / G, head = kvh * G + row % G;
  const int q0 = p.cu_q[seq], qlen = p.cu_q[seq + 1] - q0;
  const bool ok = row0 + r16 < sg.n * G && qlen > 0;
  w.load_q(0, p.q + (int64_t)(ok ? q0 + qlen - 1 : 0) * p.sqt + (int64_t)head * p.sqh, ok);
  const int keys = sg.chunks * ATT_CHUNK;  // every one of them exists
  w.qpos[0] = keys - 1;
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
  int wave, c0, cstep;    // position i of the walk is block i % 4 of chunk c0 + cstep (i / 4)
  int pg_cache, pg_base;  // SRC_FAST: page ids of this wavefront's tile for 64 positions from pg_base, one per lane

  __device__ __forceinline__ int key_at(int i) const { return (c0 + cstep * (i >> 2)) * ATT_CHUNK + (i & 3) * ATT_BLOCK + 16 * wave; }
  __device__ __forceinline__ void init(const AttnParams& p, int seq, int kvh, int keys, const uint8_t* lds, int wave_, int c0_, int cstep_) {
    src = make_source<KIND>(p, seq, kvh, 0, keys);
    wave = wave_;
    c0 = c0_;
    cstep = cstep_;
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
  __device__ __forceinline__ void issue(int i, int stage) {
    const int key0 = key_at(i);
    const uint32_t dst = lds0 + stage * SPL_STAGE;
    if constexpr (KIND == SRC_FAST) {
      if (i - pg_base >= 64) {  // wave-uniform
        pg_base = i;
        pg_cache = src.bt[min(key_at(i + (int)(threadIdx.x & 63)), src.last) >> src.shift];
      }
      const int pg = __builtin_amdgcn_readlane(pg_cache, i - pg_base), off = key0 & (src.ps - 1);
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

// Query rows lr0 .. lr0 + 16 TILES - 1 of a group and kv head as MFMA operands.
template <int TILES>
__device__ __forceinline__ void shared_load_queries(const AttnParams& p, const SharedGroup& sg, int kvh, int lr0, uint4 (&qf)[TILES][4]) {
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const int G = p.Hq / p.Hkv, rows = sg.n * G;
#pragma unroll
  for (int t = 0; t < TILES; t++) {
    const int lr = lr0 + 16 * t + r16;
    const int row = min(lr, rows - 1);
    const int seq = sg.seq0 + row / G, head = kvh * G + row % G;
    const int q0 = p.cu_q[seq], qlen = p.cu_q[seq + 1] - q0;
    const bool ok = lr < rows && qlen > 0;
    const bf16_t* qp = p.q + (int64_t)(ok ? q0 + qlen - 1 : 0) * p.sqt + (int64_t)head * p.sqh + 8 * g;
#pragma unroll
    for (int s = 0; s < 4; s++) qf[t][s] = ldg16(qp + 32 * s, ok);
  }
}

// One 64-key block from its LDS stage (keys, then values, laid out as attn_prefill_lds_kernel has them): scores, online
// softmax and P V of TILES 16-row tiles.
template <class ET, int TILES>
__device__ __forceinline__ void shared_block_compute(const uint8_t* ks, float scale, const uint4 (&qf)[TILES][4], float (&m)[TILES],
                                                   float (&l)[TILES], f32x4 (&acc)[TILES][8]) {
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
      for (int t = 0; t < TILES; t++) st[t][tt] = ET::mfma(kfr, qf[t][s], st[t][tt]);
    }
  uint4 pf[TILES][2];
#pragma unroll
  for (int t = 0; t < TILES; t++)
    attn_softmax_tile<ET>(st[t], 0, scale, 0, m[t], l[t], acc[t], pf[t], true);  // every key is visible
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
      for (int t = 0; t < TILES; t++) acc[t][f] = ET::mfma(vf, pf[t][ch], acc[t][f]);
    }
}

// Launch 1 for heads of 128: the chunk's keys and values are shared by the workgroup through LDS: 4 wavefronts with TILES
// 16-row tiles each, 64-key blocks brought in by direct-to-LDS loads into one of two 32 KB stages (two workgroups on a
// CU cover each other's waits), operands, softmax and P V as in attn_prefill_lds_kernel (same layouts and swizzles, same
// bits). Every wavefront loads the 16 keys of one tile of the block. A chunk is read once per 64 TILES query rows.
template <class ET, int TILES, int QT, int KIND>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void attn_shared_chunks_lds_kernel(AttnParams p, SharedParams sp) {
  const int index = shared_kind(sp);
  if (index < 0) {
    attn_own_chunks<ET, 128, 128, QT, KIND, 4, false>(p, sp, -1 - index);
    return;
  }
  constexpr int D = 128, KS = D / 32, RB = 64 * TILES;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * SPL_STAGE];
  int kvh, chunk, place;
  const int G = p.Hq / p.Hkv;
  SharedGroup sg;
  if (!shared_unit(p, sp, index, RB, sg, place, kvh, chunk)) return;
  const int rows = sg.n * G, row0 = place * RB;
  if (chunk >= sg.chunks || row0 >= rows) return;  // uniform over the block
  constexpr int nb = ATT_CHUNK / ATT_BLOCK;
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int keys = sg.chunks * ATT_CHUNK;  // every one of them exists

  const int mine = min(sp.cpw, (sg.chunks - chunk + 7) >> 3), n = nb * mine;  // chunks, blocks of this workgroup
  SharedLoader<KIND> ld;
  ld.init(p, sg.src, kvh, keys, lds, wave, chunk, 8);
  ld.issue(0, 0);
  ld.issue(1, 1);

  // ---- this wavefront's query tiles
  uint4 qf[TILES][KS];
  shared_load_queries<TILES>(p, sg, kvh, row0 + 16 * wave * TILES, qf);
  const bool any = row0 + 16 * wave * TILES < rows;  // wave-uniform: a wavefront without rows only loads
  for (int c = 0; c < mine; c++) {
    float m[TILES], l[TILES];
    f32x4 acc[TILES][8];
#pragma unroll
    for (int t = 0; t < TILES; t++) {
      m[t] = -INFINITY;
      l[t] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int b = 0; b < nb; b++) {
      const int i = c * nb + b;
      // 8 loads per block and wavefront, the youngest of which are those of the next block (or the last chunk's stores,
      // which are younger still and make the wait stronger): at most 8 outstanding means that block i has landed
      if (i + 1 < n) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (any) shared_block_compute<ET, TILES>(lds + (b & 1) * SPL_STAGE, p.qk_scale, qf, m, l, acc);
      __syncthreads();  // everyone has read the stage
      if (i + 2 < n) ld.issue(i + 2, b & 1);
    }
    // lane (r16 = query row, g) holds dims 16 f + 4 g .. + 3 of fragment f
#pragma unroll
    for (int t = 0; t < TILES; t++) {
      const int lr = row0 + 16 * (wave * TILES + t);
      if (lr + r16 >= rows) continue;
      float* image = sp.shared_part + (((int64_t)(sg.tile0 + (lr >> 4)) * p.Hkv + kvh) * sp.max_chunks + chunk + 8 * c) * sp.shared_floats;
#pragma unroll
      for (int f = 0; f < 8; f++)
        ((float4*)image)[(4 * f + g) * 16 + r16] = make_float4(acc[t][f][0], acc[t][f][1], acc[t][f][2], acc[t][f][3]);
      if (g == 0) ((float2*)(image + D * 16))[r16] = make_float2(m[t], l[t]);
    }
  }
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
  const int ns = min(sg.chunks, max(kv_len, 0) / ATT_CHUNK);  // a sequence shorter than its group's prefix: whole chunks
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
      const float* image = sp.shared_part + ((int64_t)(sg.tile0 + (row >> 4)) * p.Hkv + kvh) * sp.max_chunks * sp.shared_floats;
      fold(image + ((int64_t)d4 * 16 + (row & 15)) * 4, image + (int64_t)4 * d4n * 16 + 2 * (row & 15), ns, sp.shared_floats);
    }
    if (nch > ns) {
      const float* image = sp.own_part + ((int64_t)seq * p.Hkv + kvh) * sp.max_own * sp.own_floats;
      fold(image + ((int64_t)d4 * G + hl) * 4, image + (int64_t)4 * d4n * G + 2 * hl, nch - ns, sp.own_floats);
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
  constexpr bool LDS = DK == 128 && DV == 128 && !PAD;
  constexpr int WAVES = LDS ? 4 : 1;
  // row tiles per wavefront: one where an average group has at most 64 rows, else two
  const int tiles = LDS && rows > 64 * (int64_t)sp.num_groups ? 2 : 1;
  const int64_t full = std::max<int64_t>(sp.num_groups, rows / (16 * WAVES * tiles)), blocks = rows / (16 * WAVES * tiles) + sp.num_groups;
  // Chunks per workgroup of the LDS form: its set-up (group, block table, queries) costs as much as two chunks, so several
  // where that leaves about 1536 workgroups (64 sequences on 32768 keys: 138 us with one chunk each, 94 with two, 103 with
  // four; 16 groups of 16: 153 / 143 / 143)
  const int64_t units = blocks * p.Hkv * sp.max_chunks;
  sp.cpw = LDS ? (int)std::max<int64_t>(1, std::min<int64_t>(16, units / 1536)) : 1;
  const int64_t swgs = sp.num_groups == 0 || sp.max_chunks == 0 ? 0 : shared_wgs(blocks, p.Hkv, sp.max_chunks, sp.cpw);
  // about 8192 wavefronts for the own chunks, at most one per chunk (16 groups of 16: 172 / 170 / 170 us with 4096 / 8192 /
  // 16384, 128 sequences in 32 groups 68 / 68 / 72)
  sp.splits = (int)std::max<int64_t>(1, std::min<int64_t>((sp.max_own + WAVES - 1) / WAVES, 8192 / (pairs * WAVES)));
  const int64_t owgs = (pairs + 7) / 8 * 8 * sp.splits;
  if (swgs + owgs > 0x7fffffff) return VX_ERR_UNSUPPORTED;
  sp.shared_sure = (int)std::min(swgs, shared_wgs(full, p.Hkv, sp.max_chunks, sp.cpw));
  sp.own_wgs = (int)owgs;
  sp.own_first = (int)((pairs + 7) / 8 * 8);
  const unsigned grid = (unsigned)(swgs + owgs);
  if constexpr (LDS) {
    if (tiles == 2) attn_shared_chunks_lds_kernel<ET, 2, QT, KIND><<<grid, 256, 0, stream>>>(p, sp);
    else attn_shared_chunks_lds_kernel<ET, 1, QT, KIND><<<grid, 256, 0, stream>>>(p, sp);
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
  // page size a power of two >= 16, and the 16 keys of a tile within SharedLoader's 32-bit offsets
  const bool fast = p.page_shift >= 4 && std::max(p.skp, p.svp) < (int64_t)1 << 27;
  if (p.Hq / p.Hkv <= 16)
    return fast ? launch_shared_prefix_t<ET, DK, DV, 1, SRC_FAST, PAD>(p, sp, stream) : launch_shared_prefix_t<ET, DK, DV, 1, SRC_GENERIC, PAD>(p, sp, stream);
  return fast ? launch_shared_prefix_t<ET, DK, DV, 2, SRC_FAST, PAD>(p, sp, stream) : launch_shared_prefix_t<ET, DK, DV, 2, SRC_GENERIC, PAD>(p, sp, stream);
}

// in translation units of their own (compile time); DKb / DVb as for launch_attn_bf16_padded
int launch_shared_prefix_bf16_padded(const AttnParams& p, const SharedParams& sp, int DKb, int DVb, hipStream_t stream);
int launch_shared_prefix_f16(const AttnParams& p, const SharedParams& sp, int DKb, int DVb, hipStream_t stream);

}  // namespace vx
