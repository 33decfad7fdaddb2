// Decode attention for groups of sequences that share the pages of a prefix (several answers to one prompt).
//   out = softmax(scale q K^T) V of one query token per sequence over its own keys, of which the first prefix_len[g]
//   lie in pages that all sequences of group g hold.
// The arithmetic is that of attn_core.h, per chunk of 256 keys at absolute positions from a fresh state, chunk states
// folded in ascending order, so the bits are those of the decode kernels on the same block tables. What changes is who
// computes a chunk state: for the whole chunks of a shared prefix the query rows of a group (its sequences times the
// query heads of a kv head) fill the matrix core's 16 columns together, and the chunk's keys are read once per tile of
// rows instead of once per sequence. The decode kernel then folds the prefix's states in front of the sequence's own
// chunks (the partly shared chunk at the prefix's end among them).
#pragma once
#include "attn_core.h"

namespace vx {

// One wavefront per (16-row tile of a group's query rows, kv head, chunk of the shared prefix). grid = (Hkv, items, chunks).
template <class ET, int DK, int DV, int KIND, bool PAD>
__device__ __forceinline__ void attn_shared_split_body(const AttnParams& p, const SharedParams& sp) {
  const int kvh = blockIdx.x, item = blockIdx.y, chunk = blockIdx.z;
  const int G = p.Hq / p.Hkv;
  const int gi = last_group_at_most(sp.num_groups, item, [&](int i) {
    return (int)((int64_t)min(max(sp.group_off[i], 0), p.num_seqs) * G / 16) + i;
  });
  if (gi < 0) return;
  const SharedGroup sg = shared_group(p, sp, gi);
  const int row0 = (item - sg.item0) * 16;
  if (chunk >= sg.chunks || row0 >= sg.n * G) return;
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;

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

  constexpr int NDV = (DV + 127) / 128;
  float4* ip = (float4*)(sp.part + (((int64_t)item * p.Hkv + kvh) * sp.max_chunks + chunk) * sp.img_floats) + lane;
  if (!ok) return;
#pragma unroll
  for (int ds = 0; ds < NDV; ds++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      if (128 * ds + 32 * g + 8 * r >= w.dv) continue;
      const int sl = (ds * 4 + r) * 2;
      ip[sl * 64] = make_float4(w.acc[0][ds * 8 + 0][r], w.acc[0][ds * 8 + 1][r], w.acc[0][ds * 8 + 2][r], w.acc[0][ds * 8 + 3][r]);
      ip[(sl + 1) * 64] = make_float4(w.acc[0][ds * 8 + 4][r], w.acc[0][ds * 8 + 5][r], w.acc[0][ds * 8 + 6][r], w.acc[0][ds * 8 + 7][r]);
    }
  ip[NDV * 8 * 64] = make_float4(w.m[0], w.l[0], 0.f, 0.f);
}
template <class ET, int DK, int DV, int KIND, bool PAD>
__global__ __launch_bounds__(64) void attn_shared_split_kernel(AttnParams p, SharedParams sp) {
  attn_shared_split_body<ET, DK, DV, KIND, PAD>(p, sp);
}

template <class ET, int DK, int DV, int QT, int KIND, int NW, bool PAD>
__global__ __launch_bounds__(64 * NW) void attn_shared_decode_kernel(AttnParams p, SharedParams sp) {
  attn_decode_fused_body<ET, DK, DV, QT, KIND, NW, PAD, true>(p, &sp);
}

template <class ET, int DK, int DV, int QT, int KIND, bool PAD>
static int launch_shared_decode(const AttnParams& p, const SharedParams& sp, hipStream_t stream) {
  // as many wavefronts per (sequence, kv head) as their chunk states have room for in LDS
  constexpr int NW = fused_lds_bytes<DV, QT, 8>() <= 160 * 1024 ? 8 : fused_lds_bytes<DV, QT, 4>() <= 160 * 1024 ? 4 : 2;
  constexpr int LDSB = fused_lds_bytes<DV, QT, NW>();
  static_assert(LDSB <= 160 * 1024, "chunk states do not fit LDS");
  static DeviceOnce once;
  const int dev = once.slot();
  if (once.need(dev)) {
    if (hipFuncSetAttribute((const void*)attn_shared_decode_kernel<ET, DK, DV, QT, KIND, NW, PAD>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, LDSB) != hipSuccess) {
      (void)hipGetLastError();
      return VX_ERR_LAUNCH;
    }
    once.mark(dev);
  }
  attn_shared_decode_kernel<ET, DK, DV, QT, KIND, NW, PAD><<<dim3(p.Hkv, p.num_seqs), 64 * NW, LDSB, stream>>>(p, sp);
  return launch_status();
}

template <class ET, int DK, int DV, bool PAD>
static int launch_shared_prefix(const AttnParams& p, const SharedParams& sp, int64_t items, hipStream_t stream) {
  const bool fast = p.page_shift >= 4;  // page size a power of two >= 16
  if (sp.num_groups > 0 && sp.max_chunks > 0) {
    const dim3 grid(p.Hkv, (unsigned)items, sp.max_chunks);
    if (fast) attn_shared_split_kernel<ET, DK, DV, SRC_FAST, PAD><<<grid, 64, 0, stream>>>(p, sp);
    else attn_shared_split_kernel<ET, DK, DV, SRC_GENERIC, PAD><<<grid, 64, 0, stream>>>(p, sp);
    const int rc = launch_status();
    if (rc != VX_OK) return rc;
  }
  if (p.Hq / p.Hkv <= 16)
    return fast ? launch_shared_decode<ET, DK, DV, 1, SRC_FAST, PAD>(p, sp, stream) : launch_shared_decode<ET, DK, DV, 1, SRC_GENERIC, PAD>(p, sp, stream);
  return fast ? launch_shared_decode<ET, DK, DV, 2, SRC_FAST, PAD>(p, sp, stream) : launch_shared_decode<ET, DK, DV, 2, SRC_GENERIC, PAD>(p, sp, stream);
}

// in translation units of their own (compile time); DKb / DVb as for launch_attn_bf16_padded
int launch_shared_prefix_bf16_padded(const AttnParams& p, const SharedParams& sp, int DKb, int DVb, int64_t items, hipStream_t stream);
int launch_shared_prefix_f16(const AttnParams& p, const SharedParams& sp, int DKb, int DVb, int64_t items, hipStream_t stream);

}  // namespace vx
