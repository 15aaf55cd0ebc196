// The C ABI (include/espetero_attn.h): argument checks, workspace carving and
// kernel selection. Nothing here allocates device memory or synchronises.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <exception>
#include <mutex>
#include <utility>
#include <vector>

#include "common.hpp"
#include "diff_math.hpp"
#include "linear_shape.hpp"
#include "logits_shape.hpp"
#include "lowrank_shape.hpp"
#include "shaped_math.hpp"

namespace esp {
hipError_t launch_stream(int dt, int HD, int NC, const KArgs& a, const PrepArgs* pa, int n_tiles, hipStream_t st);
hipError_t launch_combine(int dt, int HD, const KArgs& a, const esp_combine* jobs, int n_jobs, int n_parts, hipStream_t st);
hipError_t launch_tiled(int dt, int HD, const KArgs& a, int n_tiles, hipStream_t st);
hipError_t launch_kv_save(const esp_attn_params* p, const void* Kb, const void* Vb, void* pool, const esp_kvsave* e, int n,
                          hipStream_t st);
hipError_t launch_kv_copy_blocks(const esp_attn_params* p, void* pool, const int32_t* pairs, int n_pairs, int n_layers,
                                 uint64_t region_elems, hipStream_t st);
hipError_t launch_kv_gather(const esp_attn_params* p, const void* pool, const int32_t* blocks, int n, void* K_out,
                            void* V_out, hipStream_t st);
hipError_t launch_kv_relayout(const esp_attn_params* p, const void* src, void* dst, int to_native, int n_blocks,
                              const int32_t* ids, hipStream_t st);
hipError_t launch_chain_advance(esp_tree* trees, int n_trees, int32_t* pos, int32_t* row_table, const int32_t* blocks, int bt,
                                int ring, hipStream_t st);
hipError_t launch_vt_stage(const esp_attn_params* p, const void* Vb, void* vt, int n_rows, hipStream_t st);
hipError_t launch_attn_prep(const PrepArgs& a, int n_rows, hipStream_t st);
hipError_t launch_head_gate(int dt, const GateArgs& a, hipStream_t st);
hipError_t gate_init_attributes();
int tiled_max_rows(int HD);
hipError_t stream_init_attributes();
hipError_t tiled_init_attributes();
hipError_t tiled256_init_attributes();
hipError_t tiled512_init_attributes();
hipError_t launch_diff_stream(int dt, const DiffArgs& a, int n_tiles, hipStream_t st);
hipError_t launch_diff_tiled(int dt, const DiffArgs& a, int n_tiles, hipStream_t st);
hipError_t launch_diff_merge(int dt, const DiffArgs& a, const esp_combine* jobs, int n_jobs, int n_parts, hipStream_t st);
hipError_t diff_init_attributes();
hipError_t diff_tiled_init_attributes();
hipError_t launch_shaped_stream(int dt, int HD, const ShapedArgs& a, int n_tiles, hipStream_t st);
hipError_t launch_shaped_tiled(int dt, int HD, const ShapedArgs& a, int n_tiles, hipStream_t st);
hipError_t launch_shaped_merge(int dt, int HD, const ShapedArgs& a, const esp_combine* jobs, int n_jobs, int n_parts, hipStream_t st);
hipError_t shaped_init_attributes();
hipError_t shaped_tiled_init_attributes();
hipError_t launch_linear(int dt, const LinearArgs& a, int n_few, int n_chunked, bool split, hipStream_t st);
hipError_t linear_init_attributes();
hipError_t launch_lowrank(int dt, const LowRankArgs& a, int rows_per_tile, int n_tiles, hipStream_t st);
hipError_t launch_logits(int dt, const LogitsArgs& a, int n_rows, hipStream_t st);
hipError_t launch_history_record(const esp_logits_params* p, uint32_t* seen, int32_t* counts, const int32_t* tokens, const int32_t* slots, int n,
                                 int given, hipStream_t st);
hipError_t launch_history_clear(const esp_logits_params* p, uint32_t* seen, int32_t* counts, const int32_t* slots, int n, hipStream_t st);
}  // namespace esp

// Library-owned device memory, one copy per GPU, held until the process ends: what
// esp_attn_forward_static uses in place of a caller's workspace (partial records of split tiles, the
// transposed batch V of the tiled kernels). In host code this name is a stand-in, not a device
// address: the address comes from hipGetSymbolAddress, once per device (device_state below), and only
// that is handed to kernels.
constexpr size_t kScratchBytes = ESP_STATIC_SCRATCH_BYTES;
static __device__ __align__(256) unsigned char scratch[kScratchBytes];

namespace {

int fail(char* err, size_t errlen, int code, const char* fmt, ...) {
  if (err && errlen) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(err, errlen, fmt, ap);
    va_end(ap);
  }
  return code;
}

int hip_fail(char* err, size_t errlen, const char* what, hipError_t e) {
  return fail(err, errlen, ESP_ELAUNCH, "%s: %s", what, hipGetErrorString(e));
}

// Checks shared by every entry point. Returns 0 or an error code.
int check_params(const esp_attn_params* p, char* err, size_t errlen) {
  if (!p) return fail(err, errlen, ESP_EINVAL, "params is NULL");
  if (p->H <= 0 || p->Hkv <= 0 || p->H % p->Hkv) return fail(err, errlen, ESP_EINVAL, "H=%d Hkv=%d: H must be a positive multiple of Hkv", p->H, p->Hkv);
  if (p->head_dim != 128 && p->head_dim != 256 && p->head_dim != 512)
    return fail(err, errlen, ESP_EUNSUPPORTED, "head_dim %d (128, 256 or 512)", p->head_dim);
  if (p->dtype != ESP_F16 && p->dtype != ESP_BF16) return fail(err, errlen, ESP_EINVAL, "dtype %d", p->dtype);
  if (p->bt <= 0 || p->bt % 16) return fail(err, errlen, ESP_EINVAL, "bt %d: tokens per block must be a positive multiple of 16", p->bt);
  if (p->q_ld < p->H * p->head_dim || p->q_ld % 8) return fail(err, errlen, ESP_EINVAL, "q_ld %d", p->q_ld);
  if (p->kv_ld < p->Hkv * p->head_dim || p->kv_ld % 8) return fail(err, errlen, ESP_EINVAL, "kv_ld %d", p->kv_ld);
  if (p->kv_base % 8) return fail(err, errlen, ESP_EINVAL, "kv_base must be a multiple of 8 elements");
  if (p->window < 0 || p->ring < 0) return fail(err, errlen, ESP_EINVAL, "window / ring negative");
  if (p->gate_headwise != 0 && p->gate_headwise != 1) return fail(err, errlen, ESP_EINVAL, "gate_headwise %d (0 or 1)", p->gate_headwise);
  return ESP_OK;
}

// Which kernel family serves rows_per_tile x G packed rows: 0 none, else the
// streaming kernel's column tiles (1, 2) or -1 for the tiled kernel.
int family(const esp_attn_params* p) {
  return esp::kernel_family(p->head_dim, p->rows_per_tile, p->H / p->Hkv);
}

// What differential attention asks of a layer's parameters beyond check_params.
int check_diff(const esp_attn_params* p, char* err, size_t errlen) {
  if (int rc = check_params(p, err, errlen)) return rc;
  if (p->head_dim != esp::kDiffHD) return fail(err, errlen, ESP_EUNSUPPORTED, "head_dim %d: differential attention serves %d", p->head_dim, esp::kDiffHD);
  if (p->H % 2 || p->Hkv % 2) return fail(err, errlen, ESP_EINVAL, "H=%d Hkv=%d: heads work in pairs", p->H, p->Hkv);
  if (p->gate || p->bidi) return fail(err, errlen, ESP_EUNSUPPORTED, "differential attention takes neither a gate nor bidirectional rows");
  if (!(p->scale > 0.0f)) return fail(err, errlen, ESP_EINVAL, "scale must be positive");
  return ESP_OK;
}

// What attention with shaped scores asks of a layer's parameters beyond check_params.
int check_shaped(const esp_attn_params* p, char* err, size_t errlen) {
  if (int rc = check_params(p, err, errlen)) return rc;
  if (p->head_dim != 128 && p->head_dim != 256) return fail(err, errlen, ESP_EUNSUPPORTED, "head_dim %d: attention with shaped scores serves 128 and 256", p->head_dim);
  if (p->H / p->Hkv > 128) return fail(err, errlen, ESP_EUNSUPPORTED, "%d query heads to a KV head (at most 128)", p->H / p->Hkv);
  if (p->gate || p->bidi) return fail(err, errlen, ESP_EUNSUPPORTED, "attention with shaped scores takes neither a gate nor bidirectional rows");
  if (!(p->scale >= 0x1p-64f && p->scale <= 0x1p64f)) return fail(err, errlen, ESP_EINVAL, "scale must be positive, from 2^-64 to 2^64");
  return ESP_OK;
}

using esp::Carve;
Carve carve(const esp_attn_params* p, int n_rows, int n_parts) {
  return esp::carve_workspace(p->H, p->Hkv, p->head_dim, p->rows_per_tile, n_rows, n_parts);
}

esp::KArgs make_args(const esp_attn_params* p, const Carve& c, void* workspace, int n_rows) {
  char* ws = static_cast<char*>(workspace);
  esp::KArgs a{};
  a.parts_o = reinterpret_cast<float*>(ws + c.parts_o);
  a.parts_ml = reinterpret_cast<float*>(ws + c.parts_ml);
  a.vt_stage = reinterpret_cast<uint16_t*>(ws + c.vt_stage);
  a.gate = p->gate;
  a.gate_ld = p->gate_ld;
  a.gate_hs = p->gate_hs;
  a.gate_off = p->gate_off;
  a.gate_ds = p->gate_headwise ? 0 : 1;
  a.H = p->H;
  a.Hkv = p->Hkv;
  a.G = p->H / p->Hkv;
  a.q_ld = p->q_ld;
  a.kv_ld = p->kv_ld;
  a.bt = p->bt;
  a.window = p->window;
  a.ring = p->ring;
  a.bidi = p->bidi;
  a.R = p->rows_per_tile;
  a.cols = a.R * a.G;
  a.n_rows = n_rows;
  a.scale_log2 = p->scale * esp::kLog2e;
  a.kv_base = p->kv_base;
  return a;
}

// A pending event pair (esp_attn_time_next) belongs to the next call that could have used it, whatever becomes of
// that call: one that launches nothing or fails its checks must not leave it armed for some later launch.
struct DropPair {
  ~DropPair() { (void)esp::take_time_next(); }
};

constexpr int kMaxDevices = 64;
struct DeviceState {
  unsigned char* scratch = nullptr;  // this device's copy of `scratch`
  bool ready = false;
};
DeviceState g_dev[kMaxDevices];
std::mutex g_dev_mutex;

// State of the current device; the first call on a device looks its copy of `scratch` up and raises the
// kernels' dynamic LDS limits (both are process-wide facts of that device, neither is stream work).
int device_state(DeviceState** out, char* err, size_t errlen) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return hip_fail(err, errlen, "hipGetDevice", e);
  if (dev < 0 || dev >= kMaxDevices) return fail(err, errlen, ESP_EUNSUPPORTED, "device ordinal %d (at most %d devices)", dev, kMaxDevices);
  std::lock_guard<std::mutex> lock(g_dev_mutex);
  DeviceState& d = g_dev[dev];
  if (!d.ready) {
    void* ps = nullptr;
    if ((e = hipGetSymbolAddress(&ps, HIP_SYMBOL(scratch))) != hipSuccess) return hip_fail(err, errlen, "hipGetSymbolAddress(scratch)", e);
    if ((e = esp::stream_init_attributes()) != hipSuccess) return hip_fail(err, errlen, "hipFuncSetAttribute (streaming kernels)", e);
    if ((e = esp::tiled_init_attributes()) != hipSuccess) return hip_fail(err, errlen, "hipFuncSetAttribute (tiled kernels)", e);
    if ((e = esp::tiled256_init_attributes()) != hipSuccess) return hip_fail(err, errlen, "hipFuncSetAttribute (tiled kernels, head dim 256)", e);
    if ((e = esp::tiled512_init_attributes()) != hipSuccess) return hip_fail(err, errlen, "hipFuncSetAttribute (tiled kernels, head dim 512)", e);
    if ((e = esp::gate_init_attributes()) != hipSuccess) return hip_fail(err, errlen, "hipFuncSetAttribute (head gate)", e);
    if ((e = esp::diff_init_attributes()) != hipSuccess) return hip_fail(err, errlen, "hipFuncSetAttribute (differential attention)", e);
    if ((e = esp::diff_tiled_init_attributes()) != hipSuccess) return hip_fail(err, errlen, "hipFuncSetAttribute (tiled differential attention)", e);
    if ((e = esp::shaped_init_attributes()) != hipSuccess) return hip_fail(err, errlen, "hipFuncSetAttribute (attention with shaped scores)", e);
    if ((e = esp::shaped_tiled_init_attributes()) != hipSuccess) return hip_fail(err, errlen, "hipFuncSetAttribute (tiled attention with shaped scores)", e);
    if ((e = esp::linear_init_attributes()) != hipSuccess) return hip_fail(err, errlen, "hipFuncSetAttribute (linear attention)", e);
    d.scratch = static_cast<unsigned char*>(ps);
    d.ready = true;
  }
  *out = &d;
  return ESP_OK;
}

}  // namespace

namespace esp {
// One pending pair per calling thread: the thread that armed it is the one whose next launch takes it, so a
// second thread driving other streams neither sees nor consumes it.
static thread_local TimeNext g_time_next;
TimeNext take_time_next() {
  const TimeNext t = g_time_next;
  g_time_next = TimeNext{};
  return t;
}
}  // namespace esp

extern "C" {

int esp_attn_abi_version(void) { return ESP_ABI_VERSION; }

int esp_attn_init(int device, char* err, size_t errlen) {
  hipDeviceProp_t prop;
  hipError_t e = hipGetDeviceProperties(&prop, device);
  if (e != hipSuccess) return hip_fail(err, errlen, "hipGetDeviceProperties", e);
  if (strncmp(prop.gcnArchName, "gfx950", 6) != 0)
    return fail(err, errlen, ESP_EUNSUPPORTED, "device %d is %s; this library is built for gfx950 only", device, prop.gcnArchName);
  // Per-device set-up with that device current: the addresses of the library's own device arrays and
  // the kernels' LDS limits, so that no later call has anything but launches left to do.
  int prev = 0;
  if ((e = hipGetDevice(&prev)) != hipSuccess) return hip_fail(err, errlen, "hipGetDevice", e);
  if (prev != device && (e = hipSetDevice(device)) != hipSuccess) return hip_fail(err, errlen, "hipSetDevice", e);
  DeviceState* d = nullptr;
  const int rc = device_state(&d, err, errlen);
  if (prev != device) (void)hipSetDevice(prev);
  return rc;
}

int esp_attn_plan_hint(const esp_attn_params* p, int device, int32_t* workgroups, int32_t* groups_per_tile,
                       int32_t* max_rows, char* err, size_t errlen) {
  if (int rc = check_params(p, err, errlen)) return rc;
  if (!workgroups || !groups_per_tile || !max_rows || p->rows_per_tile <= 0)
    return fail(err, errlen, ESP_EINVAL, "NULL output or rows_per_tile <= 0");
  int cus = 0;
  hipError_t e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device);
  if (e != hipSuccess) return hip_fail(err, errlen, "hipDeviceGetAttribute", e);
  const int fam = family(p);
  // What is resident at once. The streaming kernel's planner splits a pass up to that many workgroups (a
  // second round would pay its per-workgroup set-up again); the tiled kernel's planner hands the pass's
  // workgroups to that many slots and picks the split that finishes earliest.
  *workgroups = fam > 0 ? cus * esp::stream_workgroups_per_cu(p->head_dim, fam) : cus * esp::tiled_workgroups_per_cu(p->head_dim);
  *groups_per_tile = fam > 0 ? p->Hkv : p->H;
  *max_rows = esp::tiled_max_rows(p->head_dim);
  return ESP_OK;
}

size_t esp_attn_workspace_bytes(const esp_attn_params* p, int32_t n_rows, int32_t n_parts) {
  if (!p || p->Hkv <= 0 || p->H <= 0 || p->rows_per_tile <= 0) return 0;
  return carve(p, n_rows, n_parts).total;
}

// Attention of one layer over a planned pass. workspace NULL: the library's own scratch array
// (esp_attn_forward_static), whose size is the limit.
static int forward_impl(const esp_attn_params* p, const void* Q, const void* Kb, const void* Vb, const void* kv_pool,
                        const int32_t* blocks, const int32_t* desc, const int32_t* pos, void* O, const esp_tile* tiles,
                        int32_t n_tiles, const esp_tree* trees, int32_t n_trees, const esp_combine* jobs, int32_t n_jobs,
                        int32_t n_parts, int32_t n_rows, void* workspace, size_t workspace_bytes, bool own_scratch,
                        const esp::PrepArgs* prep, void* stream, char* err, size_t errlen) {
  DropPair drop_pair;
  if (int rc = check_params(p, err, errlen)) return rc;
  if (n_tiles < 0 || n_trees < 0 || n_jobs < 0 || n_parts < 0 || n_rows < 0) return fail(err, errlen, ESP_EINVAL, "negative count");
  if (n_tiles == 0) return ESP_OK;
  if ((!prep && !Q) || !O || !tiles || !trees) return fail(err, errlen, ESP_EINVAL, "Q, O, tiles, trees must not be NULL");
  if (!prep && ((Kb == nullptr) != (Vb == nullptr))) return fail(err, errlen, ESP_EINVAL, "Kb and Vb: both, or neither (the pass's rows are read from the pool)");
  const bool rows_in_pool = !prep && !Kb;
  if (n_trees == 0) return fail(err, errlen, ESP_EINVAL, "%d tiles without trees", n_tiles);
  if (!kv_pool) return fail(err, errlen, ESP_EINVAL, "kv_pool is NULL");
  if (!p->ring && !blocks) return fail(err, errlen, ESP_EINVAL, "blocks is NULL on a layer without rings");
  if (p->window > 0 && !pos) return fail(err, errlen, ESP_EINVAL, "pos is NULL on a sliding-window layer");
  if (p->rows_per_tile <= 0) return fail(err, errlen, ESP_EINVAL, "rows_per_tile %d", p->rows_per_tile);
  if (n_jobs > 0 && !jobs) return fail(err, errlen, ESP_EINVAL, "jobs is NULL");
  if (n_jobs > 0 && n_parts == 0) return fail(err, errlen, ESP_EINVAL, "n_jobs %d without partial records", n_jobs);
  if (!(p->scale > 0.0f)) return fail(err, errlen, ESP_EINVAL, "scale must be positive");
  const int fam = family(p);
  if (fam < 0 && p->rows_per_tile > esp::tiled_max_rows(p->head_dim))
    return fail(err, errlen, ESP_EUNSUPPORTED, "rows_per_tile %d: the tiled kernel takes at most %d rows per tile at head_dim %d",
                p->rows_per_tile, esp::tiled_max_rows(p->head_dim), p->head_dim);
  if (fam > 0 && n_tiles > 65535)
    return fail(err, errlen, ESP_EUNSUPPORTED, "%d tiles in one pass: the streaming kernel's grid takes at most 65535", n_tiles);
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev, err, errlen)) return rc;
  const Carve c = carve(p, n_rows, n_parts);
  if (own_scratch) {
    if (c.total > kScratchBytes)
      return fail(err, errlen, ESP_EWORKSPACE, "this pass needs %zu bytes of scratch; the library's own array holds %zu "
                  "(use esp_attn_forward with a workspace)", c.total, kScratchBytes);
    workspace = dev->scratch;
    workspace_bytes = kScratchBytes;
  }
  if (!workspace || workspace_bytes < c.total)
    return fail(err, errlen, ESP_EWORKSPACE, "workspace %zu bytes, %zu needed", workspace_bytes, c.total);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(err, errlen, ESP_EINVAL, "workspace must be 16-byte aligned");

  hipStream_t st = static_cast<hipStream_t>(stream);
  esp::KArgs a = make_args(p, c, workspace, n_rows);
  a.Q = static_cast<const uint16_t*>(Q);
  a.Kb = static_cast<const uint16_t*>(Kb);
  a.Vb = static_cast<const uint16_t*>(Vb);
  a.pool = static_cast<const uint16_t*>(kv_pool);
  a.blocks = blocks;
  a.desc = reinterpret_cast<const int4*>(desc);
  a.pos = reinterpret_cast<const int4*>(pos);
  a.O = static_cast<uint16_t*>(O);
  a.tiles = tiles;
  a.trees = trees;

  hipError_t e;
  if (fam > 0) {
    e = esp::launch_stream(p->dtype, p->head_dim, fam, a, prep, n_tiles, st);
    if (e != hipSuccess) return hip_fail(err, errlen, "attn_stream launch", e);
  } else {
    if (n_rows > 0 && !rows_in_pool) {
      e = esp::launch_vt_stage(p, Vb, a.vt_stage, n_rows, st);
      if (e != hipSuccess) return hip_fail(err, errlen, "vt_stage launch", e);
    }
    e = esp::launch_tiled(p->dtype, p->head_dim, a, n_tiles, st);
    if (e != hipSuccess) return hip_fail(err, errlen, "attn_tiled launch", e);
  }
  if (n_jobs > 0) {
    e = esp::launch_combine(p->dtype, p->head_dim, a, jobs, n_jobs, n_parts, st);
    if (e != hipSuccess) return hip_fail(err, errlen, "attn_combine launch", e);
  }
  return ESP_OK;
}

int esp_attn_forward(const esp_attn_params* p, const void* Q, const void* Kb, const void* Vb, const void* kv_pool,
                     const int32_t* blocks, const int32_t* desc, const int32_t* pos, void* O, const esp_tile* tiles,
                     int32_t n_tiles, const esp_tree* trees, int32_t n_trees, const esp_combine* jobs, int32_t n_jobs,
                     int32_t n_parts, int32_t n_rows, void* workspace, size_t workspace_bytes, void* stream, char* err,
                     size_t errlen) {
  return forward_impl(p, Q, Kb, Vb, kv_pool, blocks, desc, pos, O, tiles, n_tiles, trees, n_trees, jobs, n_jobs, n_parts, n_rows,
                      workspace, workspace_bytes, false, nullptr, stream, err, errlen);
}

int esp_attn_forward_static(const esp_attn_params* p, const void* Q, const void* Kb, const void* Vb, const void* kv_pool,
                            const int32_t* blocks, const int32_t* desc, const int32_t* pos, void* O, const esp_tile* tiles,
                            int32_t n_tiles, const esp_tree* trees, int32_t n_trees, const esp_combine* jobs, int32_t n_jobs,
                            int32_t n_parts, int32_t n_rows, void* stream, char* err, size_t errlen) {
  return forward_impl(p, Q, Kb, Vb, kv_pool, blocks, desc, pos, O, tiles, n_tiles, trees, n_trees, jobs, n_jobs, n_parts, n_rows,
                      nullptr, 0, true, nullptr, stream, err, errlen);
}

int esp_attn_validate(const esp_attn_params* p, const esp_tile* tiles, int32_t n_tiles, const esp_tree* trees, int32_t n_trees,
                      const esp_combine* jobs, int32_t n_jobs, int32_t n_parts, int32_t n_rows, const int32_t* blocks,
                      int32_t n_block_entries, int32_t pool_blocks, char* err, size_t errlen) {
  if (int rc = check_params(p, err, errlen)) return rc;
  if (n_tiles < 0 || n_trees < 0 || n_jobs < 0 || n_parts < 0 || n_rows < 0 || n_block_entries < 0 || pool_blocks < 0)
    return fail(err, errlen, ESP_EINVAL, "negative count");
  if (p->rows_per_tile <= 0) return fail(err, errlen, ESP_EINVAL, "rows_per_tile %d", p->rows_per_tile);
  if ((n_tiles && !tiles) || (n_trees && !trees) || (n_jobs && !jobs)) return fail(err, errlen, ESP_EINVAL, "NULL record array");
  if (!p->ring && n_block_entries && !blocks) return fail(err, errlen, ESP_EINVAL, "blocks is NULL");
  const int64_t bt = p->bt;
  for (int i = 0; i < n_trees; ++i) {
    const esp_tree& t = trees[i];
    if (t.base < 0 || t.M < 0 || int64_t(t.base) + t.M > n_rows)
      return fail(err, errlen, ESP_EINVAL, "tree %d: rows [%d, %d + %d) outside the pass's %d rows", i, t.base, t.base, t.M, n_rows);
    if (t.P < 0 || t.table < 0) return fail(err, errlen, ESP_EINVAL, "tree %d: P %d, table %d", i, t.P, t.table);
    if (p->ring) {
      if (t.P > 0 && int64_t(t.table) + p->ring > pool_blocks)
        return fail(err, errlen, ESP_EINVAL, "tree %d: ring blocks [%d, %d + %d) outside the pool's %d blocks", i, t.table, t.table, p->ring, pool_blocks);
    } else {
      const int64_t nb = (t.P + bt - 1) / bt;
      if (t.table + nb > n_block_entries)
        return fail(err, errlen, ESP_EINVAL, "tree %d: block list [%d, %d + %lld) outside the %d entries of blocks", i, t.table, t.table,
                    (long long)nb, n_block_entries);
      for (int64_t b = 0; b < nb; ++b)
        if (blocks[t.table + b] < 0 || blocks[t.table + b] >= pool_blocks)
          return fail(err, errlen, ESP_EINVAL, "tree %d: block %d (entry %lld of its list) outside the pool's %d blocks", i, blocks[t.table + b],
                      (long long)b, pool_blocks);
    }
  }
  // every partial record is written by exactly one tile and read by exactly one job
  std::vector<int32_t> part_job(size_t(n_parts), -1);
  for (int j = 0; j < n_jobs; ++j) {
    const esp_combine& c = jobs[j];
    if (c.r0 < 0 || c.rows <= 0 || c.rows > p->rows_per_tile || int64_t(c.r0) + c.rows > n_rows)
      return fail(err, errlen, ESP_EINVAL, "job %d: rows [%d, %d + %d), %d rows per tile, %d rows in the pass", j, c.r0, c.r0, c.rows,
                  p->rows_per_tile, n_rows);
    if (c.part0 < 0 || c.nparts <= 0 || int64_t(c.part0) + c.nparts > n_parts)
      return fail(err, errlen, ESP_EINVAL, "job %d: parts [%d, %d + %d) outside the pass's %d records", j, c.part0, c.part0, c.nparts, n_parts);
    for (int q = c.part0; q < c.part0 + c.nparts; ++q) {
      if (part_job[size_t(q)] >= 0) return fail(err, errlen, ESP_EINVAL, "partial record %d is merged by jobs %d and %d", q, part_job[size_t(q)], j);
      part_job[size_t(q)] = j;
    }
  }
  std::vector<char> part_written(size_t(n_parts), 0);
  for (int i = 0; i < n_tiles; ++i) {
    const esp_tile& t = tiles[i];
    if (t.tree < 0 || t.tree >= n_trees) return fail(err, errlen, ESP_EINVAL, "tile %d: tree %d of %d", i, t.tree, n_trees);
    const esp_tree& tr = trees[t.tree];
    if (t.r0 < tr.base || t.r0 >= tr.base + tr.M)
      return fail(err, errlen, ESP_EINVAL, "tile %d: first row %d outside its tree's rows [%d, %d)", i, t.r0, tr.base, tr.base + tr.M);
    if ((t.r0 - tr.base) % p->rows_per_tile) return fail(err, errlen, ESP_EINVAL, "tile %d: first row %d is no multiple of %d rows into its tree", i, t.r0, p->rows_per_tile);
    const bool open = t.k1 == INT32_MAX;  // up to the tree's cached length when the kernel runs
    if (t.k0 < 0 || (!open && (t.k1 < t.k0 || t.k1 > tr.P)) || (open && t.k0 > tr.P))
      return fail(err, errlen, ESP_EINVAL, "tile %d: cached range [%d, %d) outside its tree's %d cached keys", i, t.k0, t.k1, tr.P);
    if (t.part < -1 || t.part >= n_parts) return fail(err, errlen, ESP_EINVAL, "tile %d: partial record %d of %d", i, t.part, n_parts);
    if (t.part >= 0) {
      if (part_written[size_t(t.part)]) return fail(err, errlen, ESP_EINVAL, "tile %d: partial record %d is written by another tile too", i, t.part);
      part_written[size_t(t.part)] = 1;
      if (n_jobs > 0) {
        const int j = part_job[size_t(t.part)];
        if (j < 0) return fail(err, errlen, ESP_EINVAL, "tile %d: no job merges its partial record %d", i, t.part);
        if (jobs[j].r0 != t.r0 || jobs[j].rows != (tr.base + tr.M - t.r0 < p->rows_per_tile ? tr.base + tr.M - t.r0 : p->rows_per_tile))
          return fail(err, errlen, ESP_EINVAL, "tile %d: job %d merges rows [%d, %d + %d), the tile holds rows from %d", i, j, jobs[j].r0,
                      jobs[j].r0, jobs[j].rows, t.r0);
      }
    }
    if (t.last < 0 || (t.last >= 2 && (t.last - 2 < t.b0 || t.last - 2 >= tr.M)))
      return fail(err, errlen, ESP_EINVAL, "tile %d: last %d (0: no batch keys, 1: from b0 on, e + 2: rows b0 = %d .. e of the tree's %d)", i, t.last,
                  t.b0, tr.M);
    if (t.b0 < 0 || t.b0 > tr.M) return fail(err, errlen, ESP_EINVAL, "tile %d: first batch key %d of %d rows", i, t.b0, tr.M);
    if (t.pad != 0 && t.pad - 1 != tr.table) return fail(err, errlen, ESP_EINVAL, "tile %d: pad %d is neither 0 nor 1 + its tree's table %d", i, t.pad, tr.table);
  }
  if (n_jobs > 0)
    for (int q = 0; q < n_parts; ++q)
      if (part_job[size_t(q)] >= 0 && !part_written[size_t(q)])
        return fail(err, errlen, ESP_EINVAL, "job %d merges partial record %d, which no tile writes", part_job[size_t(q)], q);
  return ESP_OK;
}

int esp_attn_validate_for(const esp_attn_params* p, int32_t mode, const esp_tile* tiles, int32_t n_tiles, const esp_tree* trees,
                          int32_t n_trees, const esp_combine* jobs, int32_t n_jobs, int32_t n_parts, int32_t n_rows, const int32_t* blocks,
                          int32_t n_block_entries, int32_t pool_blocks, char* err, size_t errlen) {
  if (int rc = esp_attn_validate(p, tiles, n_tiles, trees, n_trees, jobs, n_jobs, n_parts, n_rows, blocks, n_block_entries, pool_blocks,
                                 err, errlen))
    return rc;
  if (mode & ~(ESP_PASS_FUSED | ESP_PASS_ROWS_IN_POOL | ESP_PASS_DIFF | ESP_PASS_SHAPED)) return fail(err, errlen, ESP_EINVAL, "mode %d", mode);
  if (mode & ESP_PASS_DIFF) {
    if (mode != ESP_PASS_DIFF) return fail(err, errlen, ESP_EINVAL, "mode %d: a pass of differential attention has no other form", mode);
    if (int rc = check_diff(p, err, errlen)) return rc;
    if (!esp::diff_family(p->rows_per_tile, p->H / p->Hkv))
      return fail(err, errlen, ESP_EUNSUPPORTED, "rows_per_tile %d (see esp_attn_diff_rows)", p->rows_per_tile);
  }
  if (mode & ESP_PASS_SHAPED) {
    if (mode != ESP_PASS_SHAPED) return fail(err, errlen, ESP_EINVAL, "mode %d: a pass of attention with shaped scores has no other form", mode);
    if (int rc = check_shaped(p, err, errlen)) return rc;
    if (!esp::shaped_family(p->head_dim, p->rows_per_tile, p->H / p->Hkv))
      return fail(err, errlen, ESP_EUNSUPPORTED, "rows_per_tile %d (see esp_attn_shaped_rows)", p->rows_per_tile);
  }
  if (mode & (ESP_PASS_DIFF | ESP_PASS_SHAPED)) {
    for (int i = 0; i < n_tiles; ++i) {
      const esp_tile& t = tiles[i];
      const int32_t P = trees[t.tree].P, k1 = std::min(t.k1, P);
      if (t.last && k1 > t.k0 && (k1 != P || t.b0 != 0))
        return fail(err, errlen, ESP_EINVAL, "tile %d: cached keys [%d, %d) and rows from %d on of a tree with %d cached keys do not meet", i, t.k0, k1, t.b0, P);
    }
  }
  if (mode & ESP_PASS_FUSED) {
    if (p->head_dim == 512 || p->rows_per_tile > 4 || family(p) <= 0)
      return fail(err, errlen, ESP_EUNSUPPORTED, "rows_per_tile %d at head_dim %d: the fused decode takes trees of 1 to 4 rows on the streaming kernel, head dim 128 or 256",
                  p->rows_per_tile, p->head_dim);
    // The fused kernel prepares the rows of its own tile only and reads a tree's batch keys from that tile's LDS
    // area: a tree is one tile group, whose first row is the tree's first row.
    for (int i = 0; i < n_trees; ++i)
      if (trees[i].M > p->rows_per_tile)
        return fail(err, errlen, ESP_EINVAL, "tree %d: %d rows; a fused pass takes trees of at most rows_per_tile = %d rows", i, trees[i].M,
                    p->rows_per_tile);
    for (int i = 0; i < n_tiles; ++i)
      if (tiles[i].r0 != trees[tiles[i].tree].base)
        return fail(err, errlen, ESP_EINVAL, "tile %d: first row %d is not its tree's first row %d (a fused pass has one tile group per tree)", i,
                    tiles[i].r0, trees[tiles[i].tree].base);
  }
  if (mode & (ESP_PASS_ROWS_IN_POOL | ESP_PASS_DIFF | ESP_PASS_SHAPED)) {
    // Row j of a tree is read at position P + j of the tree's own block list (or ring).
    const int64_t bt = p->bt;
    for (int i = 0; i < n_trees; ++i) {
      const esp_tree& t = trees[i];
      if (t.M == 0) continue;
      if ((mode & ESP_PASS_ROWS_IN_POOL) && family(p) < 0 && (t.P - t.base) % 16)
        return fail(err, errlen, ESP_EINVAL, "tree %d: P %d - base %d is no multiple of 16: the tiled kernel reads a pass's rows from the pool in "
                    "16-token sub-blocks (pass Kb / Vb for this pass)", i, t.P, t.base);
      if (p->ring) {
        if (int64_t(t.table) + p->ring > pool_blocks)
          return fail(err, errlen, ESP_EINVAL, "tree %d: ring blocks [%d, %d + %d) outside the pool's %d blocks", i, t.table, t.table, p->ring, pool_blocks);
        if (t.M > int64_t(p->ring) * bt - p->window + 1)
          return fail(err, errlen, ESP_EINVAL, "tree %d: %d rows appended to a ring of %d x %lld tokens overwrite keys that its first rows still see "
                      "(window %d): pass Kb / Vb for this pass", i, t.M, p->ring, (long long)bt, p->window);
      } else {
        const int64_t nb = (int64_t(t.P) + t.M + bt - 1) / bt;
        if (t.table + nb > n_block_entries)
          return fail(err, errlen, ESP_EINVAL, "tree %d: block list [%d, %d + %lld) with its own rows appended lies outside the %d entries of blocks", i,
                      t.table, t.table, (long long)nb, n_block_entries);
        for (int64_t b = (int64_t(t.P) + bt - 1) / bt; b < nb; ++b)
          if (blocks[t.table + b] < 0 || blocks[t.table + b] >= pool_blocks)
            return fail(err, errlen, ESP_EINVAL, "tree %d: block %d (entry %lld of its list) outside the pool's %d blocks", i, blocks[t.table + b],
                        (long long)b, pool_blocks);
      }
    }
  }
  return ESP_OK;
}

int esp_attn_time_next(void* start_event, void* stop_event) {
  if ((start_event == nullptr) != (stop_event == nullptr)) return ESP_EINVAL;
  esp::g_time_next.start = static_cast<hipEvent_t>(start_event);
  esp::g_time_next.stop = static_cast<hipEvent_t>(stop_event);
  return ESP_OK;
}

int esp_attn_combine(const esp_attn_params* p, void* O, const esp_combine* jobs, int32_t n_jobs, int32_t n_parts,
                     int32_t n_rows, void* workspace, size_t workspace_bytes, void* stream, char* err, size_t errlen) {
  if (int rc = check_params(p, err, errlen)) return rc;
  if (n_jobs < 0 || n_parts < 0 || n_rows < 0) return fail(err, errlen, ESP_EINVAL, "negative count");
  if (n_jobs == 0) return ESP_OK;
  if (!O || !jobs) return fail(err, errlen, ESP_EINVAL, "O and jobs must not be NULL");
  if (n_parts == 0) return fail(err, errlen, ESP_EINVAL, "n_jobs %d without partial records", n_jobs);
  if (p->rows_per_tile <= 0) return fail(err, errlen, ESP_EINVAL, "rows_per_tile %d", p->rows_per_tile);
  const Carve c = carve(p, n_rows, n_parts);
  if (!workspace || workspace_bytes < c.total)
    return fail(err, errlen, ESP_EWORKSPACE, "workspace %zu bytes, %zu needed", workspace_bytes, c.total);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(err, errlen, ESP_EINVAL, "workspace must be 16-byte aligned");
  esp::KArgs a = make_args(p, c, workspace, n_rows);
  a.O = static_cast<uint16_t*>(O);
  hipError_t e = esp::launch_combine(p->dtype, p->head_dim, a, jobs, n_jobs, n_parts, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ESP_OK : hip_fail(err, errlen, "attn_combine launch", e);
}

int esp_kv_save(const esp_attn_params* p, const void* Kb, const void* Vb, void* kv_pool, const esp_kvsave* entries,
                int32_t n_entries, void* stream, char* err, size_t errlen) {
  if (int rc = check_params(p, err, errlen)) return rc;
  if (n_entries < 0) return fail(err, errlen, ESP_EINVAL, "n_entries negative");
  if (n_entries == 0) return ESP_OK;
  if (!Kb || !Vb || !kv_pool || !entries) return fail(err, errlen, ESP_EINVAL, "NULL argument");
  hipError_t e = esp::launch_kv_save(p, Kb, Vb, kv_pool, entries, n_entries, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ESP_OK : hip_fail(err, errlen, "kv_save launch", e);
}

int esp_kv_copy_blocks(const esp_attn_params* p, void* kv_pool, const int32_t* pairs, int32_t n_pairs, int32_t n_layers,
                       uint64_t region_elems, void* stream, char* err, size_t errlen) {
  if (int rc = check_params(p, err, errlen)) return rc;
  if (n_pairs < 0 || n_layers < 0) return fail(err, errlen, ESP_EINVAL, "negative count");
  if (n_pairs == 0 || n_layers == 0) return ESP_OK;
  if (!kv_pool || !pairs) return fail(err, errlen, ESP_EINVAL, "NULL argument");
  if (region_elems % 8) return fail(err, errlen, ESP_EINVAL, "region_elems must be a multiple of 8");
  hipError_t e = esp::launch_kv_copy_blocks(p, kv_pool, pairs, n_pairs, n_layers, region_elems, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ESP_OK : hip_fail(err, errlen, "kv_copy_blocks launch", e);
}

int esp_kv_gather(const esp_attn_params* p, const void* kv_pool, const int32_t* blocks, int32_t n_tokens, void* K_out,
                  void* V_out, void* stream, char* err, size_t errlen) {
  if (int rc = check_params(p, err, errlen)) return rc;
  if (n_tokens < 0) return fail(err, errlen, ESP_EINVAL, "n_tokens negative");
  if (n_tokens == 0) return ESP_OK;
  if (!kv_pool || !blocks || !K_out || !V_out) return fail(err, errlen, ESP_EINVAL, "NULL argument");
  hipError_t e = esp::launch_kv_gather(p, kv_pool, blocks, n_tokens, K_out, V_out, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ESP_OK : hip_fail(err, errlen, "kv_gather launch", e);
}

int esp_kv_relayout(const esp_attn_params* p, const void* src_pool, int32_t src_layout, void* dst_pool, int32_t dst_layout,
                    int32_t n_blocks, void* stream, char* err, size_t errlen) {
  if (int rc = check_params(p, err, errlen)) return rc;
  if (n_blocks < 0) return fail(err, errlen, ESP_EINVAL, "n_blocks negative");
  if (!((src_layout == ESP_LAYOUT_REFERENCE && dst_layout == ESP_LAYOUT_NATIVE) ||
        (src_layout == ESP_LAYOUT_NATIVE && dst_layout == ESP_LAYOUT_REFERENCE)))
    return fail(err, errlen, ESP_EINVAL, "layouts %d -> %d: one side reference, the other native", src_layout, dst_layout);
  if (n_blocks == 0) return ESP_OK;
  if (!src_pool || !dst_pool) return fail(err, errlen, ESP_EINVAL, "NULL argument");
  hipError_t e = esp::launch_kv_relayout(p, src_pool, dst_pool, dst_layout == ESP_LAYOUT_NATIVE, n_blocks, nullptr,
                                         static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ESP_OK : hip_fail(err, errlen, "kv_relayout launch", e);
}

int esp_kv_export_blocks(const esp_attn_params* p, const void* kv_pool, const int32_t* blocks, int32_t n_blocks, void* out,
                         void* stream, char* err, size_t errlen) {
  if (int rc = check_params(p, err, errlen)) return rc;
  if (n_blocks < 0) return fail(err, errlen, ESP_EINVAL, "n_blocks negative");
  if (n_blocks == 0) return ESP_OK;
  if (!kv_pool || !blocks || !out) return fail(err, errlen, ESP_EINVAL, "NULL argument");
  hipError_t e = esp::launch_kv_relayout(p, static_cast<const uint16_t*>(kv_pool) + p->kv_base, out, 0, n_blocks, blocks,
                                         static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ESP_OK : hip_fail(err, errlen, "kv_export_blocks launch", e);
}

int esp_kv_import_blocks(const esp_attn_params* p, const void* in, const int32_t* blocks, int32_t n_blocks, void* kv_pool,
                         void* stream, char* err, size_t errlen) {
  if (int rc = check_params(p, err, errlen)) return rc;
  if (n_blocks < 0) return fail(err, errlen, ESP_EINVAL, "n_blocks negative");
  if (n_blocks == 0) return ESP_OK;
  if (!kv_pool || !blocks || !in) return fail(err, errlen, ESP_EINVAL, "NULL argument");
  hipError_t e = esp::launch_kv_relayout(p, in, static_cast<uint16_t*>(kv_pool) + p->kv_base, 1, n_blocks, blocks,
                                         static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ESP_OK : hip_fail(err, errlen, "kv_import_blocks launch", e);
}

int esp_chain_advance(esp_tree* trees, int32_t n_trees, int32_t* pos, int32_t* row_table, const int32_t* blocks, int32_t bt,
                      int32_t ring, void* stream, char* err, size_t errlen) {
  if (n_trees < 0) return fail(err, errlen, ESP_EINVAL, "negative count");
  if (n_trees == 0) return ESP_OK;
  if (!trees || !pos) return fail(err, errlen, ESP_EINVAL, "trees and pos must not be NULL");
  if (bt <= 0 || bt % 16) return fail(err, errlen, ESP_EINVAL, "bt %d: tokens per block must be a positive multiple of 16", bt);
  if (ring < 0) return fail(err, errlen, ESP_EINVAL, "ring negative");
  if (row_table && !ring && !blocks) return fail(err, errlen, ESP_EINVAL, "blocks is NULL on a layer without rings");
  const hipError_t e = esp::launch_chain_advance(trees, n_trees, pos, row_table, blocks, bt, ring, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(err, errlen, "chain_advance launch", e);
  return ESP_OK;
}

int esp_head_gate(const esp_gate_params* p, void* O, const void* X, const void* Wg, float* dots, int32_t n_rows,
                  void* stream, char* err, size_t errlen) {
  if (!p) return fail(err, errlen, ESP_EINVAL, "params is NULL");
  if (p->H <= 0 || p->H > 64) return fail(err, errlen, p->H <= 0 ? ESP_EINVAL : ESP_EUNSUPPORTED, "H=%d (1 .. 64)", p->H);
  if (p->head_dim <= 0 || p->head_dim % 8 || p->head_dim > 1024)
    return fail(err, errlen, ESP_EINVAL, "head_dim %d: a multiple of 8, at most 1024", p->head_dim);
  if (p->D <= 0 || p->D % 8) return fail(err, errlen, ESP_EINVAL, "D %d: a positive multiple of 8", p->D);
  if (p->dtype != ESP_F16 && p->dtype != ESP_BF16) return fail(err, errlen, ESP_EINVAL, "dtype %d", p->dtype);
  if (p->x_ld < p->D || p->x_ld % 8) return fail(err, errlen, ESP_EINVAL, "x_ld %d", p->x_ld);
  if (O && (p->q_ld < p->H * p->head_dim || p->q_ld % 8)) return fail(err, errlen, ESP_EINVAL, "q_ld %d", p->q_ld);
  if (n_rows < 0) return fail(err, errlen, ESP_EINVAL, "negative count");
  if (!O && !dots) return fail(err, errlen, ESP_EINVAL, "neither O nor dots");
  if (n_rows == 0) return ESP_OK;
  if (!X || !Wg) return fail(err, errlen, ESP_EINVAL, "X and Wg must not be NULL");
  int shift = -1;
  for (int s = 3; s <= 10; ++s)
    if (p->head_dim == 1 << s) shift = s;
  esp::GateArgs a{static_cast<uint16_t*>(O), static_cast<const uint16_t*>(X), static_cast<const uint16_t*>(Wg), dots,
                  n_rows, p->H, p->head_dim, shift, p->D, p->q_ld, p->x_ld};
  if (!O) {  // the dots kernel has an LDS limit to raise; in place nothing needs the set-up
    DeviceState* d = nullptr;
    if (int rc = device_state(&d, err, errlen)) return rc;
  }
  const hipError_t e = esp::launch_head_gate(p->dtype, a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(err, errlen, "head_gate launch", e);
  return ESP_OK;
}

// Checks of esp_prep_params shared by esp_attn_prep and esp_attn_decode_fused.
static int check_prep(const esp_prep_params* p, bool with_table, const void* kv_pool, char* err, size_t errlen) {
  if (!p) return fail(err, errlen, ESP_EINVAL, "params is NULL");
  if (p->H <= 0 || p->Hkv <= 0) return fail(err, errlen, ESP_EINVAL, "H=%d Hkv=%d", p->H, p->Hkv);
  if (p->head_dim != 128 && p->head_dim != 256 && p->head_dim != 512)
    return fail(err, errlen, ESP_EUNSUPPORTED, "head_dim %d (128, 256 or 512)", p->head_dim);
  if (p->dtype != ESP_F16 && p->dtype != ESP_BF16) return fail(err, errlen, ESP_EINVAL, "dtype %d", p->dtype);
  const int HD = p->head_dim;
  if (p->x_ld % 4 || p->q_off % 4 || p->q_hs % 4 || p->k_off % 4 || p->v_off % 4 || p->q_off < 0 || p->k_off < 0 || p->v_off < 0)
    return fail(err, errlen, ESP_EINVAL, "x_ld, q_off, q_hs, k_off, v_off must be non-negative multiples of 4 floats");
  if (p->q_hs < HD) return fail(err, errlen, ESP_EINVAL, "q_hs %d < head_dim", p->q_hs);
  if (p->x_ld < p->q_off + (p->H - 1) * p->q_hs + HD || p->x_ld < p->k_off + p->Hkv * HD || p->x_ld < p->v_off + p->Hkv * HD)
    return fail(err, errlen, ESP_EINVAL, "x_ld %d does not hold the q / k / v columns", p->x_ld);
  if (p->q_ld < p->H * HD || p->q_ld % 4 || p->kv_ld < p->Hkv * HD || p->kv_ld % 4)
    return fail(err, errlen, ESP_EINVAL, "q_ld %d / kv_ld %d", p->q_ld, p->kv_ld);
  if (HD == 512 && (p->q_ld % 8 || p->kv_ld % 8)) return fail(err, errlen, ESP_EINVAL, "q_ld %d / kv_ld %d: multiples of 8 at head_dim 512", p->q_ld, p->kv_ld);
  const int rd = p->rope_dims, rd_min = HD == 512 ? 16 : 8;  // as the header states them: half of rope_dims in whole chunks of a lane's 4 dims; of 8 (and strides of 8) at head_dim 512, which this kernel does not need
  if (rd < 0 || rd > HD || (rd != 0 && (rd < rd_min || (rd & (rd - 1)))))
    return fail(err, errlen, ESP_EINVAL, "rope_dims %d: 0 or a power of two in [%d, head_dim]", rd, rd_min);
  if (with_table) {
    if (!kv_pool) return fail(err, errlen, ESP_EINVAL, "row_table without kv_pool");
    if (p->bt <= 0 || p->bt % 16) return fail(err, errlen, ESP_EINVAL, "bt %d: tokens per block must be a positive multiple of 16", p->bt);
    if (p->kv_base % 8) return fail(err, errlen, ESP_EINVAL, "kv_base must be a multiple of 8 elements");
  }
  return ESP_OK;
}

int esp_attn_prep(const esp_prep_params* p, const float* X, const float* qn_w, const float* kn_w, const int32_t* pos,
                  const float* inv_freq, const int32_t* rope_sel, void* Q, void* Kb, void* Vb, const int32_t* row_table,
                  void* kv_pool, int32_t n_rows, void* stream, char* err, size_t errlen) {
  DropPair drop_pair;
  if (int rc = check_prep(p, row_table != nullptr, kv_pool, err, errlen)) return rc;
  if (n_rows < 0) return fail(err, errlen, ESP_EINVAL, "negative count");
  if (n_rows == 0) return ESP_OK;
  if (!X || !qn_w || !kn_w || !Q) return fail(err, errlen, ESP_EINVAL, "X, qn_w, kn_w, Q must not be NULL");
  if ((!Kb || !Vb) && (Kb || Vb || !row_table))
    return fail(err, errlen, ESP_EINVAL, "Kb and Vb may be left out together, and only with a row_table (the rows then live in the pool alone)");
  if (p->rope_dims > 0 && (!pos || !inv_freq)) return fail(err, errlen, ESP_EINVAL, "pos and inv_freq must not be NULL when dims rotate");
  esp::PrepArgs a{X, qn_w, kn_w, reinterpret_cast<const int4*>(pos), inv_freq, rope_sel, static_cast<uint16_t*>(Q),
                  static_cast<uint16_t*>(Kb), static_cast<uint16_t*>(Vb), reinterpret_cast<const int4*>(row_table),
                  static_cast<uint16_t*>(kv_pool), *p};
  const hipError_t e = esp::launch_attn_prep(a, n_rows, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(err, errlen, "attn_prep launch", e);
  return ESP_OK;
}

int esp_attn_decode_fused(const esp_prep_params* pp, const esp_attn_params* p, const float* X, const float* qn_w, const float* kn_w,
                          const int32_t* pos, const float* inv_freq, const int32_t* rope_sel, const int32_t* row_table,
                          void* kv_pool, const int32_t* blocks, const int32_t* desc, void* O, const esp_tile* tiles,
                          int32_t n_tiles, const esp_tree* trees, int32_t n_trees, const esp_combine* jobs, int32_t n_jobs,
                          int32_t n_parts, int32_t n_rows, void* workspace, size_t workspace_bytes, void* stream, char* err,
                          size_t errlen) {
  if (int rc = check_prep(pp, row_table != nullptr, kv_pool, err, errlen)) return rc;
  if (int rc = check_params(p, err, errlen)) return rc;
  if (pp->H != p->H || pp->Hkv != p->Hkv || pp->head_dim != p->head_dim || pp->dtype != p->dtype)
    return fail(err, errlen, ESP_EINVAL, "the prep and the attention parameters name different heads, head dims or element types");
  if (row_table && (pp->bt != p->bt || pp->kv_base != p->kv_base))
    return fail(err, errlen, ESP_EINVAL, "the prep and the attention parameters name different pool regions or block sizes");
  if (p->head_dim == 512) return fail(err, errlen, ESP_EUNSUPPORTED, "the fused decode serves head dims 128 and 256");
  if (p->rows_per_tile <= 0 || p->rows_per_tile > 4 || family(p) <= 0)
    return fail(err, errlen, ESP_EUNSUPPORTED, "rows_per_tile %d: the fused decode takes trees of 1 to 4 rows, one tile each, on the streaming kernel",
                p->rows_per_tile);
  if (n_tiles > 0 && (!X || !qn_w || !kn_w)) return fail(err, errlen, ESP_EINVAL, "X, qn_w, kn_w must not be NULL");
  if (pp->rope_dims > 0 && (!pos || !inv_freq)) return fail(err, errlen, ESP_EINVAL, "pos and inv_freq must not be NULL when dims rotate");
  if (!pos) return fail(err, errlen, ESP_EINVAL, "pos is NULL");
  const esp::PrepArgs a{X, qn_w, kn_w, reinterpret_cast<const int4*>(pos), inv_freq, rope_sel, nullptr, nullptr, nullptr,
                        reinterpret_cast<const int4*>(row_table), static_cast<uint16_t*>(kv_pool), *pp};
  return forward_impl(p, nullptr, nullptr, nullptr, kv_pool, blocks, desc, pos, O, tiles, n_tiles, trees, n_trees, jobs, n_jobs, n_parts,
                      n_rows, workspace, workspace_bytes, false, &a, stream, err, errlen);
}

// ---- differential attention ------------------------------------------------------
int32_t esp_attn_diff_rows(const esp_attn_params* p, int32_t rows) {
  if (check_diff(p, nullptr, 0) != ESP_OK || rows <= 0) return 0;
  return esp::diff_rows(rows, p->H / p->Hkv);
}

int esp_attn_diff_hint(const esp_attn_params* p, int device, int32_t* workgroups, int32_t* groups_per_tile, char* err, size_t errlen) {
  if (int rc = check_diff(p, err, errlen)) return rc;
  const int fam = esp::diff_family(p->rows_per_tile, p->H / p->Hkv);
  if (!workgroups || !groups_per_tile) return fail(err, errlen, ESP_EINVAL, "NULL output");
  if (!fam) return fail(err, errlen, ESP_EUNSUPPORTED, "rows_per_tile %d (see esp_attn_diff_rows)", p->rows_per_tile);
  int cus = 0;
  const hipError_t e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device);
  if (e != hipSuccess) return hip_fail(err, errlen, "hipDeviceGetAttribute", e);
  *workgroups = cus * esp::diff_workgroups_per_cu(fam);
  *groups_per_tile = p->Hkv / 2;
  return ESP_OK;
}

size_t esp_attn_diff_workspace_bytes(const esp_attn_params* p, int32_t n_parts) {
  if (!p || p->Hkv <= 0 || p->H <= 0 || p->rows_per_tile <= 0) return 0;
  return esp::carve_diff(p->H, p->rows_per_tile, n_parts).total;
}

int esp_attn_diff(const esp_attn_params* p, const esp_diff_params* d, const void* Q, const void* kv_pool, const int32_t* blocks, void* O,
                  const esp_tile* tiles, int32_t n_tiles, const esp_tree* trees, int32_t n_trees, const esp_combine* jobs, int32_t n_jobs,
                  int32_t n_parts, int32_t n_rows, void* workspace, size_t workspace_bytes, void* stream, char* err, size_t errlen) {
  if (int rc = check_diff(p, err, errlen)) return rc;
  if (!d || !d->weight) return fail(err, errlen, ESP_EINVAL, "the pairs' weights must not be NULL");
  if (d->norm_w && !(d->eps >= 0.0f)) return fail(err, errlen, ESP_EINVAL, "eps must not be negative");
  if (n_tiles < 0 || n_trees < 0 || n_jobs < 0 || n_parts < 0 || n_rows < 0) return fail(err, errlen, ESP_EINVAL, "negative count");
  if (n_tiles == 0) return ESP_OK;
  if (!Q || !O || !tiles || !trees || !kv_pool) return fail(err, errlen, ESP_EINVAL, "Q, O, tiles, trees, kv_pool must not be NULL");
  if (n_trees == 0 || n_rows == 0) return fail(err, errlen, ESP_EINVAL, "%d tiles without trees or rows", n_tiles);
  if (!p->ring && !blocks) return fail(err, errlen, ESP_EINVAL, "blocks is NULL on a layer without rings");
  if (n_jobs > 0 && !jobs) return fail(err, errlen, ESP_EINVAL, "jobs is NULL");
  if ((n_jobs > 0) != (n_parts > 0)) return fail(err, errlen, ESP_EINVAL, "%d merge jobs with %d partial records", n_jobs, n_parts);
  const int fam = esp::diff_family(p->rows_per_tile, p->H / p->Hkv);
  if (!fam) return fail(err, errlen, ESP_EUNSUPPORTED, "rows_per_tile %d (see esp_attn_diff_rows)", p->rows_per_tile);
  if (n_tiles > 65535 || n_jobs > 65535) return fail(err, errlen, ESP_EUNSUPPORTED, "%d tiles, %d jobs in one pass: at most 65535", n_tiles, n_jobs);
  const esp::DiffCarve c = esp::carve_diff(p->H, p->rows_per_tile, n_parts);
  if (n_parts > 0 && (!workspace || workspace_bytes < c.total))
    return fail(err, errlen, ESP_EWORKSPACE, "workspace %zu bytes, %zu needed", workspace ? workspace_bytes : size_t(0), c.total);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(err, errlen, ESP_EINVAL, "workspace must be 16-byte aligned");
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev, err, errlen)) return rc;
  esp::DiffArgs a{};
  a.Q = static_cast<const uint16_t*>(Q);
  a.pool = static_cast<const uint16_t*>(kv_pool);
  a.blocks = blocks;
  a.O = static_cast<uint16_t*>(O);
  a.tiles = tiles;
  a.trees = trees;
  a.parts_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + c.parts_o);
  a.parts_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + c.parts_ml);
  a.weight = d->weight;
  a.norm_w = d->norm_w;
  a.H = p->H;
  a.Hkv = p->Hkv;
  a.G = p->H / p->Hkv;
  a.q_ld = p->q_ld;
  a.bt = p->bt;
  a.window = p->window;
  a.ring = p->ring;
  a.R = p->rows_per_tile;
  a.cols = a.R * a.G;
  a.scale_log2 = p->scale * esp::kLog2e;
  a.eps = d->eps;
  a.factor = d->factor;
  a.kv_base = p->kv_base;
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e = fam > 0 ? esp::launch_diff_stream(p->dtype, a, n_tiles, st) : esp::launch_diff_tiled(p->dtype, a, n_tiles, st);
  if (e != hipSuccess) return hip_fail(err, errlen, "attn_diff launch", e);
  if (n_jobs > 0) {
    e = esp::launch_diff_merge(p->dtype, a, jobs, n_jobs, n_parts, st);
    if (e != hipSuccess) return hip_fail(err, errlen, "attn_diff_merge launch", e);
  }
  return ESP_OK;
}

// ---- attention with shaped scores ------------------------------------------------
int32_t esp_attn_shaped_rows(const esp_attn_params* p, int32_t rows) {
  if (check_shaped(p, nullptr, 0) != ESP_OK || rows <= 0) return 0;
  return esp::shaped_rows(rows, p->H / p->Hkv);
}

int esp_attn_shaped_hint(const esp_attn_params* p, int device, int32_t* workgroups, int32_t* groups_per_tile, char* err, size_t errlen) {
  if (int rc = check_shaped(p, err, errlen)) return rc;
  const int fam = esp::shaped_family(p->head_dim, p->rows_per_tile, p->H / p->Hkv);
  if (!workgroups || !groups_per_tile) return fail(err, errlen, ESP_EINVAL, "NULL output");
  if (!fam) return fail(err, errlen, ESP_EUNSUPPORTED, "rows_per_tile %d (see esp_attn_shaped_rows)", p->rows_per_tile);
  int cus = 0;
  const hipError_t e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device);
  if (e != hipSuccess) return hip_fail(err, errlen, "hipDeviceGetAttribute", e);
  *workgroups = cus * esp::shaped_workgroups_per_cu(p->head_dim, fam);
  *groups_per_tile = p->Hkv;
  return ESP_OK;
}

size_t esp_attn_shaped_workspace_bytes(const esp_attn_params* p, int32_t n_parts) {
  if (!p || p->Hkv <= 0 || p->H <= 0 || p->head_dim <= 0 || p->rows_per_tile <= 0) return 0;
  return esp::carve_shaped(p->H, p->head_dim, p->rows_per_tile, n_parts).total;
}

int esp_attn_shaped(const esp_attn_params* p, const esp_shape_params* shape, const void* Q, const void* kv_pool, const int32_t* blocks, void* O,
                    const esp_tile* tiles, int32_t n_tiles, const esp_tree* trees, int32_t n_trees, const esp_combine* jobs, int32_t n_jobs,
                    int32_t n_parts, int32_t n_rows, void* workspace, size_t workspace_bytes, void* stream, char* err, size_t errlen) {
  if (int rc = check_shaped(p, err, errlen)) return rc;
  if (!shape) return fail(err, errlen, ESP_EINVAL, "shape is NULL");
  if (!(shape->cap >= 0.0f) || (shape->cap > 0.0f && !(shape->cap >= p->scale * 0x1p-60f && shape->cap <= 0x1p120f)))
    return fail(err, errlen, ESP_EINVAL, "cap must be 0, or from 2^-60 of the scale to 2^120");
  if (n_tiles < 0 || n_trees < 0 || n_jobs < 0 || n_parts < 0 || n_rows < 0) return fail(err, errlen, ESP_EINVAL, "negative count");
  if (n_tiles == 0) return ESP_OK;
  if (!Q || !O || !tiles || !trees || !kv_pool) return fail(err, errlen, ESP_EINVAL, "Q, O, tiles, trees, kv_pool must not be NULL");
  if (n_trees == 0 || n_rows == 0) return fail(err, errlen, ESP_EINVAL, "%d tiles without trees or rows", n_tiles);
  if (!p->ring && !blocks) return fail(err, errlen, ESP_EINVAL, "blocks is NULL on a layer without rings");
  if (n_jobs > 0 && !jobs) return fail(err, errlen, ESP_EINVAL, "jobs is NULL");
  if ((n_jobs > 0) != (n_parts > 0)) return fail(err, errlen, ESP_EINVAL, "%d merge jobs with %d partial records", n_jobs, n_parts);
  const int fam = esp::shaped_family(p->head_dim, p->rows_per_tile, p->H / p->Hkv);
  if (!fam) return fail(err, errlen, ESP_EUNSUPPORTED, "rows_per_tile %d (see esp_attn_shaped_rows)", p->rows_per_tile);
  if (n_tiles > 65535 || n_jobs > 65535) return fail(err, errlen, ESP_EUNSUPPORTED, "%d tiles, %d jobs in one pass: at most 65535", n_tiles, n_jobs);
  const esp::DiffCarve c = esp::carve_shaped(p->H, p->head_dim, p->rows_per_tile, n_parts);
  if (n_parts > 0 && (!workspace || workspace_bytes < c.total))
    return fail(err, errlen, ESP_EWORKSPACE, "workspace %zu bytes, %zu needed", workspace ? workspace_bytes : size_t(0), c.total);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(err, errlen, ESP_EINVAL, "workspace must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(shape->spans) % 8 || reinterpret_cast<uintptr_t>(shape->slopes) % 4)
    return fail(err, errlen, ESP_EINVAL, "spans must be 8-byte, slopes 4-byte aligned");
  if ((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(kv_pool)) % 16 || reinterpret_cast<uintptr_t>(O) % 8)
    return fail(err, errlen, ESP_EINVAL, "Q and kv_pool must be 16-byte, O 8-byte aligned");
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev, err, errlen)) return rc;
  esp::ShapedArgs a{};
  a.Q = static_cast<const uint16_t*>(Q);
  a.pool = static_cast<const uint16_t*>(kv_pool);
  a.blocks = blocks;
  a.O = static_cast<uint16_t*>(O);
  a.tiles = tiles;
  a.trees = trees;
  a.parts_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + c.parts_o);
  a.parts_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + c.parts_ml);
  a.slopes = shape->slopes;
  a.spans = reinterpret_cast<const int2*>(shape->spans);
  a.H = p->H;
  a.Hkv = p->Hkv;
  a.G = p->H / p->Hkv;
  a.q_ld = p->q_ld;
  a.bt = p->bt;
  a.window = p->window;
  a.ring = p->ring;
  a.R = p->rows_per_tile;
  a.cols = a.R * a.G;
  a.scale_log2 = shape->cap > 0.0f ? float(2.0 * double(p->scale) * 1.4426950408889634 / double(shape->cap)) : p->scale * esp::kLog2e;
  a.cap_log2 = shape->cap * esp::kLog2e;
  if (shape->cap > 0.0f) {
    // Behind |z| = t the terms from i on are more than 2^-25 of the sum: where a cap is so far from the scale that fp32 does not hold their
    // coefficients, the polynomial ends in front of them (huge caps), or is not used (tiny ones).
    constexpr double kTanh[5] = {0.9999996972994237, -0.33330212938002485, 0.13281112912937199, -0.050836244052251026, 0.013773716642020806};
    constexpr double kUntil[5] = {0.0, 3e-4, 0.021, 0.09, 0.19};
    const double z = double(p->scale) / double(shape->cap);
    double power = double(p->scale) * 1.4426950408889634, until = 0.7;
    int terms = 0;
    for (; terms < 5; ++terms, power *= z * z) {
      const double c = kTanh[terms] * power;
      if (std::fabs(c) > FLT_MAX) until = 0.0;
      if (std::fabs(c) > FLT_MAX || std::fabs(c) < FLT_MIN) break;
      a.tanh_c[terms] = float(c);
    }
    if (terms < 5) until = std::min(until, kUntil[terms]);
    a.tanh_below = float(std::min(until / z, double(FLT_MAX)));
    if (terms == 5) {
      constexpr double kShort[3] = {0.9999998947913661, -0.33328590898156374, 0.13015407522207817};
      power = double(p->scale) * 1.4426950408889634;
      for (int i = 0; i < 3; ++i, power *= z * z) a.tanh_s[i] = float(kShort[i] * power);
      a.tanh_short = float(0.2 / z);
    }
  }
  a.kv_base = p->kv_base;
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e = fam > 0 ? esp::launch_shaped_stream(p->dtype, p->head_dim, a, n_tiles, st) : esp::launch_shaped_tiled(p->dtype, p->head_dim, a, n_tiles, st);
  if (e != hipSuccess) return hip_fail(err, errlen, "attn_shaped launch", e);
  if (n_jobs > 0) {
    e = esp::launch_shaped_merge(p->dtype, p->head_dim, a, jobs, n_jobs, n_parts, st);
    if (e != hipSuccess) return hip_fail(err, errlen, "attn_shaped_merge launch", e);
  }
  return ESP_OK;
}

// ---- low-rank adapters -------------------------------------------------------------
static int check_lowrank(const esp_lowrank_params* p, char* err, size_t errlen) {
  if (!p) return fail(err, errlen, ESP_EINVAL, "params is NULL");
  if (p->dtype != ESP_F16 && p->dtype != ESP_BF16) return fail(err, errlen, ESP_EINVAL, "dtype %d", p->dtype);
  if (p->D <= 0 || p->D % 8) return fail(err, errlen, ESP_EINVAL, "D %d: a positive multiple of 8", p->D);
  if (p->rank <= 0 || p->rank % 8 || p->rank > esp::kLowRankMost)
    return fail(err, errlen, ESP_EINVAL, "rank %d: a positive multiple of 8, at most %d", p->rank, esp::kLowRankMost);
  if (p->n_slices < 1 || p->n_slices > ESP_LOWRANK_SLICES) return fail(err, errlen, ESP_EINVAL, "n_slices %d (1 to %d)", p->n_slices, int(ESP_LOWRANK_SLICES));
  if (p->n_adapters <= 0) return fail(err, errlen, ESP_EINVAL, "n_adapters %d", p->n_adapters);
  if (p->x_ld < p->D || p->x_ld % 8) return fail(err, errlen, ESP_EINVAL, "x_ld %d", p->x_ld);
  int64_t blocks = 0, out = 0;
  for (int s = 0; s < p->n_slices; ++s) {
    if (p->width[s] <= 0 || p->y_off[s] < 0 || int64_t(p->y_off[s]) + p->width[s] > p->y_ld)
      return fail(err, errlen, ESP_EINVAL, "slice %d: columns [%d, %d + %d) of a row of %d", s, p->y_off[s], p->y_off[s], p->width[s], p->y_ld);
    for (int q = 0; q < s; ++q)
      if (p->y_off[s] < p->y_off[q] + p->width[q] && p->y_off[q] < p->y_off[s] + p->width[s])
        return fail(err, errlen, ESP_EINVAL, "slices %d and %d overlap", q, s);
    blocks += (int64_t(p->width[s]) + 255) / 256;
    out += p->width[s];
  }
  if (blocks > 65535 || out > INT32_MAX) return fail(err, errlen, ESP_EUNSUPPORTED, "%lld columns in the slices", (long long)out);
  return ESP_OK;
}

int32_t esp_lowrank_rows(const esp_lowrank_params* p, int32_t n_rows) {
  if (check_lowrank(p, nullptr, 0) != ESP_OK || n_rows <= 0) return 0;
  return esp::lowrank_rows(n_rows);
}

size_t esp_lowrank_workspace_bytes(const esp_lowrank_params* p, int32_t n_tiles, int32_t n_slots) {
  if (check_lowrank(p, nullptr, 0) != ESP_OK || n_tiles <= 0 || n_slots <= 0) return 0;
  return esp::lowrank_workspace(*p, n_slots);
}

int esp_lowrank_add(const esp_lowrank_params* p, const void* X, const void* A, const void* B, const float* scale, float* Y, const int32_t* order,
                    int32_t n_slots, const esp_lowrank_tile* tiles, int32_t n_tiles, void* workspace, size_t workspace_bytes, void* stream,
                    char* err, size_t errlen) {
  if (int rc = check_lowrank(p, err, errlen)) return rc;
  if (n_slots < 0 || n_tiles < 0) return fail(err, errlen, ESP_EINVAL, "negative count");
  if (p->rows_per_tile != 16 && p->rows_per_tile != 64) return fail(err, errlen, ESP_EUNSUPPORTED, "rows_per_tile %d (see esp_lowrank_rows)", p->rows_per_tile);
  if (n_tiles == 0) return ESP_OK;
  if (n_tiles > 65535) return fail(err, errlen, ESP_EUNSUPPORTED, "%d tiles (at most 65535)", n_tiles);
  int64_t columns = 0;  // in blocks of 128
  for (int s = 0; s < p->n_slices; ++s) columns += (int64_t(p->width[s]) + 127) / 128;
  if ((int64_t(n_tiles) + 7) / 8 * 8 * columns >= 1 << 24)
    return fail(err, errlen, ESP_EUNSUPPORTED, "%d tiles of %lld blocks of columns: more workgroups than a launch has", n_tiles, (long long)columns);
  if (n_slots == 0) return fail(err, errlen, ESP_EINVAL, "%d tiles without rows", n_tiles);
  if (!X || !A || !B || !scale || !Y || !order || !tiles) return fail(err, errlen, ESP_EINVAL, "X, A, B, scale, Y, order, tiles must not be NULL");
  if ((reinterpret_cast<uintptr_t>(X) | reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B) | reinterpret_cast<uintptr_t>(workspace)) % 16)
    return fail(err, errlen, ESP_EINVAL, "X, A, B and the workspace must be 16-byte aligned");
  const size_t need = esp::lowrank_workspace(*p, n_slots);
  if (!workspace || workspace_bytes < need) return fail(err, errlen, ESP_EWORKSPACE, "workspace %zu bytes, %zu needed", workspace ? workspace_bytes : size_t(0), need);
  esp::LowRankArgs a{};
  a.X = static_cast<const uint16_t*>(X);
  a.A = static_cast<const uint16_t*>(A);
  a.B = static_cast<const uint16_t*>(B);
  a.scale = scale;
  a.Y = Y;
  a.order = order;
  a.tiles = tiles;
  a.low = static_cast<float*>(workspace);
  a.D = p->D;
  a.rank = p->rank;
  a.n_slices = p->n_slices;
  a.n_low = p->n_slices * p->rank;
  a.x_ld = p->x_ld;
  a.y_ld = p->y_ld;
  a.n_slots = n_slots;
  a.splits = esp::lowrank_splits(p->D, a.n_low, p->rows_per_tile, n_tiles);
  a.chunk = esp::lowrank_chunk(p->D, a.splits);
  for (int s = 0; s < p->n_slices; ++s) {
    a.y_off[s] = p->y_off[s];
    a.width[s] = p->width[s];
    a.n_out += p->width[s];
  }
  const hipError_t e = esp::launch_lowrank(p->dtype, a, p->rows_per_tile, n_tiles, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ESP_OK : hip_fail(err, errlen, "lowrank launch", e);
}

int esp_lowrank_validate(const esp_lowrank_params* p, const int32_t* order, int32_t n_slots, const esp_lowrank_tile* tiles, int32_t n_tiles,
                         int32_t n_rows, char* err, size_t errlen) {
  if (int rc = check_lowrank(p, err, errlen)) return rc;
  if (n_slots < 0 || n_tiles < 0 || n_rows < 0) return fail(err, errlen, ESP_EINVAL, "negative count");
  if ((n_slots && !order) || (n_tiles && !tiles)) return fail(err, errlen, ESP_EINVAL, "order or tiles is NULL");
  if (p->rows_per_tile != 16 && p->rows_per_tile != 64) return fail(err, errlen, ESP_EUNSUPPORTED, "rows_per_tile %d (see esp_lowrank_rows)", p->rows_per_tile);
  std::vector<std::pair<int32_t, int32_t>> rows;  // and the tile that names each
  try {
    for (int32_t i = 0; i < n_tiles; ++i) {
      const esp_lowrank_tile& t = tiles[i];
      if (t.adapter < 0 || t.adapter >= p->n_adapters) return fail(err, errlen, ESP_EINVAL, "tile %d: adapter %d of %d", i, t.adapter, p->n_adapters);
      if (t.count < 0 || t.count > p->rows_per_tile) return fail(err, errlen, ESP_EINVAL, "tile %d: %d rows, rows_per_tile is %d", i, t.count, p->rows_per_tile);
      if (t.first < 0 || int64_t(t.first) + t.count > n_slots)
        return fail(err, errlen, ESP_EINVAL, "tile %d: slots [%d, %d + %d) of %d", i, t.first, t.first, t.count, n_slots);
      for (int32_t s = t.first; s < t.first + t.count; ++s) {
        if (order[s] < 0 || order[s] >= n_rows) return fail(err, errlen, ESP_EINVAL, "tile %d: row %d of %d", i, order[s], n_rows);
        rows.emplace_back(order[s], i);
      }
      if (rows.size() > size_t(n_rows)) break;  // one of them comes twice
    }
    std::sort(rows.begin(), rows.end());
  } catch (const std::exception& e) {
    return fail(err, errlen, ESP_EINVAL, "%s", e.what());
  }
  for (size_t i = 1; i < rows.size(); ++i)
    if (rows[i].first == rows[i - 1].first)
      return fail(err, errlen, ESP_EINVAL, "tile %d: row %d is named twice (also by tile %d)", rows[i].second, rows[i].first, rows[i - 1].second);
  return ESP_OK;
}

// ---- logits ------------------------------------------------------------------------
static int check_logits(const esp_logits_params* p, char* err, size_t errlen) {
  if (!p) return fail(err, errlen, ESP_EINVAL, "params is NULL");
  if (p->dtype != ESP_F16 && p->dtype != ESP_BF16 && p->dtype != ESP_F32) return fail(err, errlen, ESP_EINVAL, "dtype %d", p->dtype);
  if (p->vocab <= 0 || p->vocab > INT32_MAX - 65536) return fail(err, errlen, ESP_EINVAL, "vocab %d", p->vocab);
  if (p->n_slots < 0 || p->n_masks < 0 || p->n_bias < 0 || p->n_bias > INT32_MAX - 65536)
    return fail(err, errlen, ESP_EINVAL, "%d slots, %d masks, %d bias entries", p->n_slots, p->n_masks, p->n_bias);
  return ESP_OK;
}

size_t esp_logits_workspace_bytes(const esp_logits_params* p, int32_t n_rows) {
  if (check_logits(p, nullptr, 0) != ESP_OK || n_rows <= 0) return 0;
  return esp::logits_workspace(p->vocab, n_rows);
}

int esp_logits_process(const esp_logits_params* p, const void* logits, float* out, int32_t* tokens, const esp_logits_row* rows, int32_t n_rows,
                       const int32_t* bias_tokens, const float* bias_values, const uint32_t* masks, uint32_t* seen, int32_t* counts,
                       int32_t record, void* workspace, size_t workspace_bytes, void* stream, char* err, size_t errlen) {
  if (int rc = check_logits(p, err, errlen)) return rc;
  if (n_rows < 0 || n_rows > 65535) return fail(err, errlen, ESP_EINVAL, "%d rows (at most 65535)", n_rows);
  if (n_rows == 0) return ESP_OK;
  if (!logits || !rows || (!out && !tokens)) return fail(err, errlen, ESP_EINVAL, "logits, rows and one of out and tokens must not be NULL");
  if (p->in_ld < p->vocab) return fail(err, errlen, ESP_EINVAL, "in_ld %d of a vocabulary of %d", p->in_ld, p->vocab);
  if (out && p->out_ld < p->vocab) return fail(err, errlen, ESP_EINVAL, "out_ld %d of a vocabulary of %d", p->out_ld, p->vocab);
  if (out == logits && (p->dtype != ESP_F32 || p->in_ld != p->out_ld)) return fail(err, errlen, ESP_EINVAL, "out may be the logits only where both are fp32 rows of one stride");
  if (record != 0 && record != 1) return fail(err, errlen, ESP_EINVAL, "record %d (0 or 1)", record);
  if (record && (!tokens || !p->n_slots)) return fail(err, errlen, ESP_EINVAL, "record without tokens or without slots");
  if (p->n_slots && (!seen || !counts)) return fail(err, errlen, ESP_EINVAL, "%d slots without histories", p->n_slots);
  if (p->n_masks && !masks) return fail(err, errlen, ESP_EINVAL, "masks is NULL");
  if (p->n_bias && (!bias_tokens || !bias_values)) return fail(err, errlen, ESP_EINVAL, "bias_tokens or bias_values is NULL");
  const size_t need = esp::logits_workspace(p->vocab, n_rows);
  if (!workspace || workspace_bytes < need) return fail(err, errlen, ESP_EWORKSPACE, "workspace %zu bytes, %zu needed", workspace ? workspace_bytes : size_t(0), need);
  if (reinterpret_cast<uintptr_t>(workspace) % 4) return fail(err, errlen, ESP_EINVAL, "workspace must be 4-byte aligned");
  esp::LogitsArgs a{};
  a.logits = logits;
  a.out = out;
  a.tokens = tokens;
  a.rows = rows;
  a.bias_tokens = bias_tokens;
  a.bias_values = bias_values;
  a.masks = masks;
  a.seen = seen;
  a.counts = counts;
  a.part_v = static_cast<float*>(workspace);
  a.part_t = static_cast<int32_t*>(workspace) + size_t(esp::logits_shape(p->vocab, n_rows).chunks) * size_t(n_rows);
  a.vocab = p->vocab;
  a.words = esp::logits_words(p->vocab);
  a.in_ld = p->in_ld;
  a.out_ld = p->out_ld;
  a.n_slots = p->n_slots;
  a.n_masks = p->n_masks;
  a.n_bias = p->n_bias;
  a.record = record;
  const hipError_t e = esp::launch_logits(p->dtype, a, n_rows, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ESP_OK : hip_fail(err, errlen, "logits launch", e);
}

int esp_logits_validate(const esp_logits_params* p, const esp_logits_row* rows, int32_t n_rows, const int32_t* bias_tokens, char* err,
                        size_t errlen) {
  if (int rc = check_logits(p, err, errlen)) return rc;
  if (n_rows < 0 || (n_rows && !rows) || (p->n_bias && !bias_tokens)) return fail(err, errlen, ESP_EINVAL, "rows or bias_tokens is NULL");
  for (int i = 0; i < n_rows; ++i) {
    const esp_logits_row& r = rows[i];
    if (r.slot < -1 || r.slot >= p->n_slots) return fail(err, errlen, ESP_EINVAL, "row %d: slot %d of %d", i, r.slot, p->n_slots);
    if (r.mask < -1 || r.mask >= p->n_masks) return fail(err, errlen, ESP_EINVAL, "row %d: mask %d of %d", i, r.mask, p->n_masks);
    if (!(r.repetition > 0.0f) || !std::isfinite(r.repetition) || !std::isfinite(r.frequency) || !std::isfinite(r.presence))
      return fail(err, errlen, ESP_EINVAL, "row %d: penalties %g, %g, %g", i, r.repetition, r.frequency, r.presence);
    if (r.n_bias < 0 || (r.n_bias && (r.bias0 < 0 || int64_t(r.bias0) + r.n_bias > p->n_bias)))
      return fail(err, errlen, ESP_EINVAL, "row %d: bias entries [%d, %d + %d) of %d", i, r.bias0, r.bias0, r.n_bias, p->n_bias);
    for (int32_t e = 0; e < r.n_bias; ++e) {
      const int32_t t = bias_tokens[r.bias0 + e];
      if (t < 0 || t >= p->vocab || (e && t <= bias_tokens[r.bias0 + e - 1]))
        return fail(err, errlen, ESP_EINVAL, "row %d: token %d at bias entry %d: in [0, %d), ascending, none twice", i, t, e, p->vocab);
    }
  }
  return ESP_OK;
}

static int check_history(const esp_logits_params* p, const uint32_t* seen, const int32_t* counts, const int32_t* slots, int32_t n, char* err, size_t errlen) {
  if (int rc = check_logits(p, err, errlen)) return rc;
  if (n < 0 || n > INT32_MAX - 65536) return fail(err, errlen, ESP_EINVAL, "%d entries", n);
  if (n && (!seen || !counts || !slots)) return fail(err, errlen, ESP_EINVAL, "seen, counts and slots must not be NULL");
  return ESP_OK;
}

int esp_history_record(const esp_logits_params* p, uint32_t* seen, int32_t* counts, const int32_t* tokens, const int32_t* slots, int32_t n,
                       int32_t given, void* stream, char* err, size_t errlen) {
  if (int rc = check_history(p, seen, counts, slots, n, err, errlen)) return rc;
  if (given != 0 && given != 1) return fail(err, errlen, ESP_EINVAL, "given %d (0 or 1)", given);
  if (n == 0) return ESP_OK;
  if (!tokens) return fail(err, errlen, ESP_EINVAL, "tokens is NULL");
  const hipError_t e = esp::launch_history_record(p, seen, counts, tokens, slots, n, given, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ESP_OK : hip_fail(err, errlen, "history_record launch", e);
}

int esp_history_clear(const esp_logits_params* p, uint32_t* seen, int32_t* counts, const int32_t* slots, int32_t n, void* stream, char* err,
                      size_t errlen) {
  if (int rc = check_history(p, seen, counts, slots, n, err, errlen)) return rc;
  if (n > 65535) return fail(err, errlen, ESP_EINVAL, "%d slots (at most 65535)", n);
  if (n == 0) return ESP_OK;
  const hipError_t e = esp::launch_history_clear(p, seen, counts, slots, n, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ESP_OK : hip_fail(err, errlen, "history_clear launch", e);
}

// ---- linear attention --------------------------------------------------------------
static int check_linear(const esp_linear_params* p, char* err, size_t errlen) {
  if (!p) return fail(err, errlen, ESP_EINVAL, "params is NULL");
  if (p->dtype != ESP_F16 && p->dtype != ESP_BF16) return fail(err, errlen, ESP_EINVAL, "dtype %d", p->dtype);
  if (p->Hk <= 0 || p->H <= 0 || p->H % p->Hk || p->H > 4096)
    return fail(err, errlen, ESP_EINVAL, "H=%d Hk=%d: H must be a positive multiple of Hk, at most 4096", p->H, p->Hk);
  if (!esp::linear_dims(p->dk, p->dv)) return fail(err, errlen, ESP_EUNSUPPORTED, "dk %d (64 or 128), dv %d (a multiple of 64, at most 512)", p->dk, p->dv);
  if (p->q_ld < p->Hk * p->dk || p->k_ld < p->Hk * p->dk || p->v_ld < p->H * p->dv || p->o_ld < p->H * p->dv)
    return fail(err, errlen, ESP_EINVAL, "q_ld %d, k_ld %d, v_ld %d, o_ld %d: a row has %d, %d, %d and %d elements", p->q_ld, p->k_ld, p->v_ld, p->o_ld,
                p->Hk * p->dk, p->Hk * p->dk, p->H * p->dv, p->H * p->dv);
  if ((p->q_ld | p->k_ld | p->v_ld | p->o_ld) % 8) return fail(err, errlen, ESP_EINVAL, "row strides must be multiples of 8");
  if (std::max(std::max(p->q_ld, p->k_ld), std::max(p->v_ld, p->o_ld)) > 1 << 24)  // 64 rows of it in 32 bits of bytes
    return fail(err, errlen, ESP_EUNSUPPORTED, "row strides of more than %d elements", 1 << 24);
  if (p->decay_ld != 0 && p->decay_ld < p->H) return fail(err, errlen, ESP_EINVAL, "decay_ld %d (0, or at least H = %d)", p->decay_ld, p->H);
  if (p->n_states < 0) return fail(err, errlen, ESP_EINVAL, "n_states %d", p->n_states);
  if (!std::isfinite(p->scale)) return fail(err, errlen, ESP_EINVAL, "scale is not finite");
  return ESP_OK;
}

int esp_linear_hint(const esp_linear_params* p, int device, int32_t* workgroups, char* err, size_t errlen) {
  if (int rc = check_linear(p, err, errlen)) return rc;
  if (!workgroups) return fail(err, errlen, ESP_EINVAL, "NULL output");
  int cus = 0;
  const hipError_t e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device);
  if (e != hipSuccess) return hip_fail(err, errlen, "hipDeviceGetAttribute", e);
  *workgroups = cus * esp::linear_workgroups_per_cu(p->dk, p->dv);
  return ESP_OK;
}

size_t esp_linear_workspace_bytes(const esp_linear_params* p, int32_t n_parts) {
  if (check_linear(p, nullptr, 0) != ESP_OK) return 0;
  return esp::carve_linear(p->H, p->dk, p->dv, n_parts).total;
}

int esp_linear_attn(const esp_linear_params* p, const void* Q, const void* K, const void* V, const float* decay, float* states, void* O,
                    const esp_linear_tile* tiles, int32_t n_tiles, int32_t n_few, int32_t n_parts, int32_t n_rows, void* workspace,
                    size_t workspace_bytes, void* stream, char* err, size_t errlen) {
  if (int rc = check_linear(p, err, errlen)) return rc;
  if (n_tiles < 0 || n_few < 0 || n_few > n_tiles || n_parts < 0 || n_rows < 0) return fail(err, errlen, ESP_EINVAL, "counts");
  if (n_tiles == 0) return ESP_OK;
  if (!tiles) return fail(err, errlen, ESP_EINVAL, "tiles must not be NULL");
  if ((n_rows > 0 || n_few < n_tiles) && (!Q || !K || !V || !O || !decay))  // (without rows states are copied or cleared)
    return fail(err, errlen, ESP_EINVAL, "Q, K, V, O and decay must not be NULL");
  if (p->n_states > 0 && !states) return fail(err, errlen, ESP_EINVAL, "states is NULL");
  if ((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V) | reinterpret_cast<uintptr_t>(O) |
       reinterpret_cast<uintptr_t>(states) | reinterpret_cast<uintptr_t>(workspace)) % 16)
    return fail(err, errlen, ESP_EINVAL, "Q, K, V, O, states and workspace must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(decay) % 4) return fail(err, errlen, ESP_EINVAL, "decay must be 4-byte aligned");
  if (n_few > 65535 || n_tiles - n_few > 65535) return fail(err, errlen, ESP_EUNSUPPORTED, "%d and %d tiles in one pass: at most 65535 of each kind", n_few, n_tiles - n_few);
  const esp::LinearCarve c = esp::carve_linear(p->H, p->dk, p->dv, n_parts);
  if (n_parts > 0 && (!workspace || workspace_bytes < c.total))
    return fail(err, errlen, ESP_EWORKSPACE, "workspace %zu bytes, %zu needed", workspace ? workspace_bytes : size_t(0), c.total);
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev, err, errlen)) return rc;
  esp::LinearArgs a{};
  a.Q = static_cast<const uint16_t*>(Q);
  a.K = static_cast<const uint16_t*>(K);
  a.V = static_cast<const uint16_t*>(V);
  a.decay = decay;
  a.states = states;
  a.O = static_cast<uint16_t*>(O);
  a.tiles = tiles;
  a.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + c.states);
  a.part_totals = reinterpret_cast<double*>(static_cast<char*>(workspace) + c.totals);
  a.H = p->H;
  a.group = p->H / p->Hk;
  a.dk = p->dk;
  a.dv = p->dv;
  a.q_ld = p->q_ld;
  a.k_ld = p->k_ld;
  a.v_ld = p->v_ld;
  a.o_ld = p->o_ld;
  a.decay_ld = p->decay_ld;
  a.scale = p->scale;
  const hipError_t e = esp::launch_linear(p->dtype, a, n_few, n_tiles - n_few, n_parts > 0, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? ESP_OK : hip_fail(err, errlen, "linear_attn launch", e);
}

int esp_linear_validate(const esp_linear_params* p, const esp_linear_tile* tiles, int32_t n_tiles, int32_t n_few, int32_t n_parts, int32_t n_rows,
                        char* err, size_t errlen) {
  if (int rc = check_linear(p, err, errlen)) return rc;
  if (n_tiles < 0 || n_few < 0 || n_few > n_tiles || n_parts < 0 || n_rows < 0) return fail(err, errlen, ESP_EINVAL, "counts");
  if (n_tiles && !tiles) return fail(err, errlen, ESP_EINVAL, "NULL record array");
  try {
    std::vector<char> row(size_t(n_rows), 0), part(size_t(n_parts), 0);
    std::vector<int32_t> writer(size_t(p->n_states), -1), reader(size_t(p->n_states), -1);  // sequences, named by their first tile
    int first = 0;
    for (int i = 0; i < n_tiles; ++i) {
      const esp_linear_tile& t = tiles[i];
      if (t.rows < 0 || t.row0 < 0 || int64_t(t.row0) + t.rows > n_rows)
        return fail(err, errlen, ESP_EINVAL, "tile %d: rows [%d, %d + %d) outside the pass's %d rows", i, t.row0, t.row0, t.rows, n_rows);
      if (i < n_few && t.rows > esp::kLinearFew) return fail(err, errlen, ESP_EINVAL, "tile %d: %d rows among those of few (at most %d)", i, t.rows, esp::kLinearFew);
      for (int r = t.row0; r < t.row0 + t.rows; ++r)
        if (row[size_t(r)]++) return fail(err, errlen, ESP_EINVAL, "tile %d: row %d is in another tile too", i, r);
      if (t.src < -1 || t.src >= p->n_states || t.dst < -1 || t.dst >= p->n_states)
        return fail(err, errlen, ESP_EINVAL, "tile %d: slots %d and %d of %d", i, t.src, t.dst, p->n_states);
      if (t.before < 0 || t.after < 0 || t.part < -1) return fail(err, errlen, ESP_EINVAL, "tile %d: segments or record negative", i);
      if ((t.before > 0 || t.after > 0) != (t.part >= 0) || (t.part >= 0 && i < n_few))
        return fail(err, errlen, ESP_EINVAL, "tile %d: %d segments in front, %d behind, first record %d", i, t.before, t.after, t.part);
      if (t.part >= 0 && int64_t(t.part) + t.before + t.after + 1 > n_parts)
        return fail(err, errlen, ESP_EINVAL, "tile %d: records [%d, %d + %d) of %d", i, t.part, t.part, t.before + t.after + 1, n_parts);
      if (t.before == 0) {
        first = i;
        if (t.src >= 0) reader[size_t(t.src)] = reader[size_t(t.src)] == -1 || reader[size_t(t.src)] == i ? i : -2;
        for (int q = t.part; t.part >= 0 && q <= t.part + t.after; ++q)
          if (part[size_t(q)]++) return fail(err, errlen, ESP_EINVAL, "tile %d: record %d is another sequence's too", i, q);
      } else {
        const esp_linear_tile& u = tiles[i - 1];
        if (i == 0 || i == n_few || u.before + 1 != t.before || u.after - 1 != t.after || u.part != t.part || u.src != t.src || u.row0 + u.rows != t.row0)
          return fail(err, errlen, ESP_EINVAL, "tile %d does not go on where the one in front of it ends", i);
      }
      if (t.after > 0 && (i + 1 >= n_tiles || tiles[i + 1].before != t.before + 1))
        return fail(err, errlen, ESP_EINVAL, "tile %d: the segment behind it is missing", i);
      if (t.after > 0 && t.dst >= 0) return fail(err, errlen, ESP_EINVAL, "tile %d: dst %d in front of its sequence's end", i, t.dst);
      if (t.dst >= 0) {
        if (writer[size_t(t.dst)] != -1) return fail(err, errlen, ESP_EINVAL, "tile %d: slot %d is another sequence's too", i, t.dst);
        writer[size_t(t.dst)] = first;
      }
    }
    for (int s = 0; s < p->n_states; ++s)
      if (writer[size_t(s)] != -1 && reader[size_t(s)] != -1 && reader[size_t(s)] != writer[size_t(s)])
        return fail(err, errlen, ESP_EINVAL, "slot %d is read by another sequence than the one that leaves its state there", s);
  } catch (const std::exception& e) {
    return fail(err, errlen, ESP_EINVAL, "%s", e.what());
  }
  return ESP_OK;
}

}  // extern "C"
