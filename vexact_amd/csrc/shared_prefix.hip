// Entry point of decode attention over shared prefixes (shared_prefix.h), and the kernels for the head sizes they are
// built for exactly.
#include "shared_prefix.h"

using namespace vx;

extern "C" {

// 16-row tiles of all groups, at most
static inline int64_t shared_tiles(int64_t num_seqs, int64_t num_groups, int64_t G) { return num_seqs * G / 16 + num_groups; }

static int64_t shared_part_bytes(int64_t num_seqs, int64_t num_groups, int64_t Hq, int64_t Hkv, int64_t Dv, int64_t max_prefix_len) {
  return shared_tiles(num_seqs, num_groups, Hq / Hkv) * Hkv * (max_prefix_len / ATT_CHUNK) * shared_image_floats(16, Dv) * 4;
}

// Sizes whose workgroups, row numbers and workspace bytes stay within their types; every product is of factors bounded before.
static bool shared_sizes_ok(int64_t num_seqs, int64_t num_groups, int64_t Hq, int64_t Hkv, int64_t Dv, int64_t max_prefix_len, int64_t max_kv_len) {
  if (Dv > 256 || Hq / Hkv > 32 || num_seqs > 65535 || Hq > 65535 || num_seqs * Hq > 0x7fffffff || num_groups > 0x7fffffff || max_kv_len > 0x7fffff00)
    return false;
  const int64_t tiles = shared_tiles(num_seqs, num_groups, Hq / Hkv) * Hkv;
  return tiles <= 0x7fffffff / (max_prefix_len / ATT_CHUNK + 8) &&  // workgroups
         num_seqs * Hkv <= ((int64_t)1 << 40) / ((max_kv_len + ATT_CHUNK - 1) / ATT_CHUNK);  // own images, below 2^16 bytes each
}

int64_t vx_shared_prefix_workspace_bytes(int64_t num_seqs, int64_t num_groups, int64_t Hq, int64_t Hkv, int64_t Dv, int64_t max_prefix_len,
                                         int64_t max_kv_len) {
  if (num_seqs <= 0 || num_groups < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || Dv <= 0 || max_prefix_len < 0 || max_kv_len <= 0) return 0;
  if (!shared_sizes_ok(num_seqs, num_groups, Hq, Hkv, Dv, max_prefix_len, max_kv_len)) return 0;
  return shared_part_bytes(num_seqs, num_groups, Hq, Hkv, Dv, max_prefix_len) +
         num_seqs * Hkv * ((max_kv_len + ATT_CHUNK - 1) / ATT_CHUNK) * shared_image_floats(Hq / Hkv, Dv) * 4;
}

int vx_shared_prefix_attention(const void* q, const void* k, const void* v, void* out, const int* cu_seqlens_q,
                               const int* seqused_k, const int* block_table, const int* group_offsets, const int* prefix_lens,
                               int64_t num_seqs, int64_t num_groups, int Hq, int Hkv, int Dk, int Dv, int64_t sqt, int64_t sqh,
                               int64_t skb, int64_t skp, int64_t skh, int64_t svb, int64_t svp, int64_t svh, int64_t sot, int64_t soh,
                               int64_t bt_stride, int64_t max_pages, int page_size, float softmax_scale, int64_t max_prefix_len,
                               int dtype, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  if (!q || !k || !v || !out || !cu_seqlens_q || !seqused_k || !block_table) return VX_ERR_ARG;
  if (num_groups > 0 && (!group_offsets || !prefix_lens)) return VX_ERR_ARG;
  if (dtype != 0 && dtype != 1) return VX_ERR_UNSUPPORTED;
  if (num_seqs < 0 || num_groups < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || Dk <= 0 || Dv <= 0 || max_prefix_len < 0) return VX_ERR_ARG;
  if (page_size <= 0 || max_pages <= 0) return VX_ERR_ARG;
  if (Dk > 256 || Dv > 256 || Hq / Hkv > 32 || num_seqs > 65535 || Hq > 65535) return VX_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) % 2 != 0) return VX_ERR_ARG;
  if (num_seqs == 0) return VX_OK;
  if (max_pages > 0x7fffff00 / page_size) return VX_ERR_UNSUPPORTED;
  const int64_t max_kv = max_pages * (int64_t)page_size;
  if (max_prefix_len > max_kv) max_prefix_len = max_kv;
  if (!shared_sizes_ok(num_seqs, num_groups, Hq, Hkv, Dv, max_prefix_len, max_kv)) return VX_ERR_UNSUPPORTED;
  const int64_t shared_bytes = shared_part_bytes(num_seqs, num_groups, Hq, Hkv, Dv, max_prefix_len);
  const int64_t need = vx_shared_prefix_workspace_bytes(num_seqs, num_groups, Hq, Hkv, Dv, max_prefix_len, max_kv);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) return VX_ERR_WORKSPACE;
  // rows that 16-byte accesses cannot address go element by element
  const bool elem = (sqt | sqh | skb | skp | skh | svb | svp | svh | sot | soh | (int64_t)Dk | (int64_t)Dv) % 8 != 0 ||
                    ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) % 16 != 0;
  AttnParams p = {};
  p.dk = Dk; p.dv = Dv; p.elem = elem ? 1 : 0;
  p.q = (const bf16_t*)q; p.sqt = sqt; p.sqh = sqh;
  p.k = (const bf16_t*)k; p.skb = skb; p.skp = skp; p.skh = skh;
  p.v = (const bf16_t*)v; p.svb = svb; p.svp = svp; p.svh = svh;
  p.o = (bf16_t*)out; p.sot = sot; p.soh = soh;
  p.cu_q = cu_seqlens_q; p.seqused_k = seqused_k;
  p.block_table = block_table; p.bt_stride = bt_stride;
  p.page_size = page_size;
  p.page_shift = -1;
  if ((page_size & (page_size - 1)) == 0) {
    int s = 0;
    while ((1 << s) < page_size) s++;
    p.page_shift = s;
  }
  p.Hq = Hq; p.Hkv = Hkv; p.num_seqs = (int)num_seqs;
  p.qk_scale = softmax_scale * 1.44269504f;
  p.causal = 1;
  p.max_kv = (int)max_kv;
  SharedParams sp = {};
  sp.group_off = group_offsets; sp.prefix_len = prefix_lens;
  sp.num_groups = (int)num_groups;
  sp.max_chunks = (int)(max_prefix_len / ATT_CHUNK);
  sp.shared_part = (float*)workspace;
  sp.shared_floats = shared_image_floats(16, Dv);
  sp.own_part = (float*)((uint8_t*)workspace + shared_bytes);
  sp.own_floats = shared_image_floats(Hq / Hkv, Dv);
  sp.max_own = (int)((max_kv + ATT_CHUNK - 1) / ATT_CHUNK);
  if (!elem) {
    if (Dk == 128 && Dv == 128)
      return dtype == 0 ? launch_shared_prefix<ElemBF16, 128, 128, false>(p, sp, stream) : launch_shared_prefix<ElemF16, 128, 128, false>(p, sp, stream);
    if (Dk == 64 && Dv == 64)
      return dtype == 0 ? launch_shared_prefix<ElemBF16, 64, 64, false>(p, sp, stream) : launch_shared_prefix<ElemF16, 64, 64, false>(p, sp, stream);
  }
  const int DVb = Dv > 128 ? 256 : (Dk > 64 || Dv > 64) ? 128 : 64;
  const int DKb = (Dk > 128 || DVb == 256) ? 256 : DVb;
  return dtype == 0 ? launch_shared_prefix_bf16_padded(p, sp, DKb, DVb, stream) : launch_shared_prefix_f16(p, sp, DKb, DVb, stream);
}

}  // extern "C"
