// K9: the entry point of attention over an 8-bit paged cache.  The kernels
// (paged8_decode.cuh) are compiled by format and type in paged8_e4m3_f16.cu and
// its like.
#include "paged8_decode.cuh"

namespace {

bool rows16(const kf_tensor4& t) {
  if (!kf::aligned16(t.ptr) || t.stride[3] != 1) return false;
  for (int i = 0; i < 2; ++i)
    if (t.size[i] > 1 && t.stride[i] % 8 != 0) return false;
  return true;
}

}  // namespace

extern "C" size_t kf_paged8_decode_workspace_bytes(int64_t Hq, int64_t Hkv, int64_t D, int sm_count) {
  if (Hq <= 0 || Hkv <= 0 || D <= 0 || sm_count <= 0) return 0;
  const int rows = unit_rows(Hq / Hkv), steps = (int)((D + 15) / 16);
  return workspace_need(sm_count * blocks_per_sm(steps, rows), rows, D);
}

extern "C" int kf_paged8_decode(const kf_paged8_decode_args* args) {
  using kf::set_error;
  const char* what = "kf_paged8_decode";
  if (!args) return set_error(KF_ERR_INVALID, "%s: null arguments", what);
  const kf_tensor4 &q = args->q, &new_k = args->new_k, &new_v = args->new_v;
  const kf_paged8_cache& cache = args->cache;
  const kf_tensor4 &k_pages = cache.k_pages, &v_pages = cache.v_pages;
  if (args->dtype != KF_F16 && args->dtype != KF_BF16)
    return set_error(KF_ERR_INVALID, "%s: dtype must be fp16 or bf16", what);
  int rc = kf::check_cache8(what, cache);
  if (rc != KF_OK) return rc;
  const int64_t B = q.size[0], Hq = q.size[1], D = q.size[3], max_pages = args->max_pages;
  const int64_t pages = k_pages.size[0], Hkv = k_pages.size[1], page_size = k_pages.size[2];
  if (B <= 0 || Hq <= 0 || max_pages <= 0) return set_error(KF_ERR_INVALID, "%s: dimensions must be non-zero", what);
  if (q.size[2] != 1) return set_error(KF_ERR_INVALID, "%s: Q must hold one token per request", what);
  if (k_pages.size[3] != D) return set_error(KF_ERR_INVALID, "%s: Q/K/V head dimensions must match", what);
  if (Hq % Hkv != 0)
    return set_error(KF_ERR_INVALID, "%s: num_query_heads must be divisible by num_kv_heads", what);
  if (max_pages > 0x7fffffffLL || B > (1 << 20) || Hq > (1 << 16))
    return set_error(KF_ERR_UNSUPPORTED, "%s: tensors too large", what);
  if (!rows16(q) || !kf::aligned16(args->o))
    return set_error(KF_ERR_INVALID, "%s: tensors need a contiguous last dim and 16-byte aligned rows", what);
  if (!q.ptr || !args->o || !args->block_table || !args->lengths)
    return set_error(KF_ERR_INVALID, "%s: null data pointer", what);
  if (!isfinite((float)args->scale * kLog2e))
    return set_error(KF_ERR_INVALID, "%s: scale must be finite in single precision", what);
  const bool fused = new_k.ptr || new_v.ptr || args->slots;
  if (fused) {
    if (!new_k.ptr || !new_v.ptr || !args->slots)
      return set_error(KF_ERR_INVALID, "%s: new_k, new_v and slots go together", what);
    for (int i = 0; i < 4; ++i)
      if (new_v.size[i] != new_k.size[i])
        return set_error(KF_ERR_INVALID, "%s: new K and V shapes must match", what);
    if (new_k.size[0] != B || new_k.size[1] != Hkv || new_k.size[2] != 1 || new_k.size[3] != D)
      return set_error(KF_ERR_INVALID, "%s: new K/V must be [B, Hkv, 1, D]", what);
    if (!rows16(new_k) || !rows16(new_v))
      return set_error(KF_ERR_INVALID, "%s: new K/V rows must be 16-byte aligned", what);
  }
  kf::DeviceGuard guard(q.ptr);
  if (guard.status()) return guard.status();

  const int rows = unit_rows(Hq / Hkv);
  const Layout l = layout_of(D, k_pages, v_pages);
  Paged8Args a;
  a.q = static_cast<const uint16_t*>(q.ptr);
  a.k = static_cast<uint8_t*>(k_pages.ptr);
  a.v = static_cast<uint8_t*>(v_pages.ptr);
  a.ks_ = cache.k_scales;
  a.vs_ = cache.v_scales;
  a.block_shift = 0;
  while (((int64_t)1 << a.block_shift) < cache.scale_block) ++a.block_shift;
  // Blocks of several tokens: a new row may change how the rows before it are
  // held, which other units of this launch may be reading; so it is stored first.
  const bool inside = fused && a.block_shift == 0;
  a.nk = inside ? static_cast<const uint16_t*>(new_k.ptr) : nullptr;
  a.nv = inside ? static_cast<const uint16_t*>(new_v.ptr) : nullptr;
  a.slots = args->slots;
  a.o = static_cast<uint16_t*>(args->o);
  a.lse = args->lse;
  a.table = args->block_table;
  a.lengths = args->lengths;
  for (int i = 0; i < 2; ++i) {
    a.qs[i] = q.stride[i];
    a.nks[i] = inside ? new_k.stride[i] : 0;
    a.nvs[i] = inside ? new_v.stride[i] : 0;
    a.kss[i] = cache.k_scale_strides[i];
    a.vss[i] = cache.v_scale_strides[i];
  }
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = k_pages.stride[i];
    a.vs[i] = v_pages.stride[i];
  }
  a.table_stride = args->table_stride;
  a.B = (int)B;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.G = (int)(Hq / Hkv);
  a.D = (int)D;
  a.page_size = (uint32_t)page_size;
  a.num_pages = (uint32_t)pages;
  a.status = args->status;
  a.box = l.box;
  a.group = l.box < 16 ? 16 : l.box;
  a.scale_log2 = (float)args->scale * kLog2e;

  int64_t blocks, most;
  rc = plan_work(what, a, max_pages, rows, tile_keys(l.steps, rows), blocks_per_sm(l.steps, rows), args->workspace,
                 args->workspace_bytes, &blocks, &most);
  if (rc != KF_OK) return rc;
  // K and V as two planes of one tensor, where that describes both and a box
  // is a whole group.
  const int64_t apart = static_cast<const uint8_t*>(v_pages.ptr) - static_cast<const uint8_t*>(k_pages.ptr);
  a.paired = l.lines && l.box >= 16 && apart != 0 && (apart > 0 ? apart : -apart) < ((int64_t)1 << 39);
  for (int i = 0; i < 3; ++i) a.paired = a.paired && (k_pages.size[i] == 1 || k_pages.stride[i] == v_pages.stride[i]);
  a.k_plane = a.paired && apart < 0 ? 1 : 0;
  a.v_plane = 1 - a.k_plane;
  const int pitch = l.steps * 16, lines = l.box * pitch / 128;
  const bool swizzle = l.steps == 2 || l.steps == 4 || l.steps == 8;
  CUtensorMap mk = {}, mv = {};
  for (int w = 0; w < (!l.lines ? 0 : a.paired ? 1 : 2); ++w) {
    const kf_tensor4& pool = a.paired ? (apart > 0 ? k_pages : v_pages) : w ? v_pages : k_pages;
    kf::PageLines t;
    t.base = pool.ptr;
    t.lines = page_size * pitch / 128;
    t.line_stride = pitch == 128 ? pool.stride[2] : 128;
    t.planes = a.paired ? 2 : 1;
    t.plane_stride = apart > 0 ? apart : -apart;
    t.heads = Hkv;
    t.head_stride = pool.stride[1];
    t.pages = pages;
    t.page_stride = pool.stride[0];
    rc = kf::encode_tmap_lines(w ? &mv : &mk, t, lines, swizzle);
    if (rc != KF_OK) return rc;
  }
  if (a.paired) mv = mk;
  if (fused && !inside) {
    kf_paged8_append_args store;
    store.cache = cache;
    store.new_k = new_k;
    store.new_v = new_v;
    store.slots = args->slots;
    store.dtype = args->dtype;
    store.stream = args->stream;
    rc = kf_paged8_append(&store);
    if (rc != KF_OK) return rc;
  }
  kf::Paged8Launch launch;
  launch.args = &a;
  launch.map_k = &mk;
  launch.map_v = &mv;
  launch.steps = l.steps;
  launch.lines = l.lines;
  launch.rows = rows;
  launch.blocks = (int)blocks;
  launch.stream = static_cast<cudaStream_t>(args->stream);
  const bool bf16 = args->dtype == KF_BF16;
  if (cache.format == KF_INT8)
    rc = bf16 ? kf::paged8_launch_int8_bf16(launch) : kf::paged8_launch_int8_f16(launch);
  else
    rc = bf16 ? kf::paged8_launch_e4m3_bf16(launch) : kf::paged8_launch_e4m3_f16(launch);
  if (rc != KF_OK || most == 1) return rc;
  return launch_join(what, a, bf16, rows, blocks, launch.stream);
}
