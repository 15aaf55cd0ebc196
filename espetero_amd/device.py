"""Calls into libespetero_attn.so with torch tensors as device memory.

torch is plumbing here (allocation, streams, host<->device copies); every
computation happens behind the C ABI. There is no fallback path: a missing or
failing library raises.
"""
import ctypes as C

import numpy as np
import torch

from . import abi, host

try:
    from . import _calls  # the per-step calls, csrc/calls.cpp
except ImportError as e:
    raise abi.EspError(f"espetero_amd/_calls.so is not built (run __graft_entry__.build()): {e}") from e

_ERRLEN = 512


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(stream):
    """hipStream_t as an int. The current stream is asked for as a raw handle: torch.cuda.current_stream() builds a Stream
    object, 2.5 us of a decode step that has 8 us of GPU work."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
    return stream.cuda_stream


def init(device=0):
    err = C.create_string_buffer(_ERRLEN)
    abi.check(abi.attn_lib().esp_attn_init(device, err, _ERRLEN), err)


def to_dev(a, device="cuda"):
    """numpy array (any dtype, incl. structured records) -> device tensor of raw bytes / ints."""
    a = np.ascontiguousarray(a)
    if a.dtype.fields is not None or a.dtype == np.uint16:
        flat = a.view(np.uint8).reshape(-1)
        return torch.from_numpy(flat.copy()).to(device)
    return torch.from_numpy(a.copy()).to(device)


def plan_hint(params, device=0):
    """(workgroups resident at once, workgroups per tile) of the kernel serving `params`:
    the planner's split target and its `groups` argument."""
    return plan_hint3(params, device)[:2]


def plan_hint3(params, device=0):
    """plan_hint plus the largest rows_per_tile the tiled kernel takes at this head_dim."""
    err = C.create_string_buffer(_ERRLEN)
    n, g, r = C.c_int32(0), C.c_int32(0), C.c_int32(0)
    abi.check(abi.attn_lib().esp_attn_plan_hint(C.byref(params), device, C.byref(n), C.byref(g), C.byref(r), err, _ERRLEN), err)
    return n.value, abi.PlanGroups(g.value, params), r.value


def workspace_bytes(params, n_rows, n_parts):
    return abi.attn_lib().esp_attn_workspace_bytes(C.byref(params), n_rows, n_parts)


def forward(params, Q, Kb, Vb, pool, blocks, desc, pos, O, tiles, n_tiles, trees, n_trees, jobs, n_jobs, n_parts, n_rows,
            workspace, stream=None):
    """All tensors are device tensors (records as byte tensors). Enqueues on `stream`."""
    _calls.attn_forward(params, Q, Kb, Vb, pool, blocks, desc, pos, O, tiles, n_tiles, trees, n_trees, jobs, n_jobs, n_parts, n_rows,
                        workspace, 0 if workspace is None else workspace.nbytes, _stream(stream))


def forward_static(params, Q, Kb, Vb, pool, blocks, desc, pos, O, tiles, n_tiles, trees, n_trees, jobs, n_jobs, n_parts, n_rows,
                   stream=None):
    """forward() over the library's own scratch array: no workspace, no allocation."""
    _calls.attn_forward_static(params, Q, Kb, Vb, pool, blocks, desc, pos, O, tiles, n_tiles, trees, n_trees, jobs, n_jobs, n_parts, n_rows,
                               _stream(stream))


def validate(params, tiles, trees, jobs, n_parts, n_rows, blocks, pool_blocks, fused=False, rows_in_pool=False, diff=False, shaped=False):
    """Host-side bounds check of a pass's records (numpy arrays) before they are uploaded. Raises EspError.
    fused: the pass goes to esp_attn_decode_fused (also: one tile group per tree, trees of at most rows_per_tile rows).
    rows_in_pool: the pass runs without Kb / Vb (also: block lists that reach P + M, P - base a multiple of 16 on the tiled kernel).
    diff, shaped: the pass goes to esp_attn_diff, or esp_attn_shaped (also: block lists that reach P + M)."""
    tiles = np.ascontiguousarray(tiles, dtype=abi.TILE_DT)
    trees = np.ascontiguousarray(trees, dtype=abi.TREE_DT)
    jobs = np.ascontiguousarray(jobs, dtype=abi.COMBINE_DT)
    blocks = None if blocks is None else np.ascontiguousarray(blocks, dtype=np.int32)
    hp = lambda a: None if a is None or a.size == 0 else a.ctypes.data  # noqa: E731
    err = C.create_string_buffer(_ERRLEN)
    mode = (abi.ESP_PASS_FUSED if fused else 0) | (abi.ESP_PASS_ROWS_IN_POOL if rows_in_pool else 0) | (abi.ESP_PASS_DIFF if diff else 0) | \
        (abi.ESP_PASS_SHAPED if shaped else 0)
    rc = abi.attn_lib().esp_attn_validate_for(C.byref(params), mode, hp(tiles), len(tiles), hp(trees), len(trees), hp(jobs), len(jobs),
                                              n_parts, n_rows, hp(blocks), 0 if blocks is None else len(blocks), pool_blocks, err, _ERRLEN)
    abi.check(rc, err)


def time_next(start, stop):
    """The next forward() records its attention kernel's begin and end into these two torch events
    (created with enable_timing=True and recorded once before, so that their handles exist)."""
    rc = abi.attn_lib().esp_attn_time_next(C.c_void_p(start.cuda_event), C.c_void_p(stop.cuda_event))
    if rc != 0:
        raise abi.EspError(f"esp_attn_time_next: error {rc}")


def combine(params, O, jobs, n_jobs, n_parts, n_rows, workspace, stream=None):
    _calls.attn_combine(params, O, jobs, n_jobs, n_parts, n_rows, workspace, workspace.nbytes, _stream(stream))


def kv_save(params, Kb, Vb, pool, entries, n_entries, stream=None):
    _calls.kv_save(params, Kb, Vb, pool, entries, n_entries, _stream(stream))


def kv_copy_blocks(params, pool, pairs, n_pairs, n_layers, region_elems, stream=None):
    _calls.kv_copy_blocks(params, pool, pairs, n_pairs, n_layers, region_elems, _stream(stream))


def kv_gather(params, pool, blocks, n_tokens, K_out, V_out, stream=None):
    err = C.create_string_buffer(_ERRLEN)
    abi.check(abi.attn_lib().esp_kv_gather(C.byref(params), _ptr(pool), _ptr(blocks), n_tokens, _ptr(K_out), _ptr(V_out),
                                           _stream(stream), err, _ERRLEN), err)


def kv_relayout(params, src, src_layout, dst, dst_layout, n_blocks, stream=None):
    err = C.create_string_buffer(_ERRLEN)
    abi.check(abi.attn_lib().esp_kv_relayout(C.byref(params), _ptr(src), src_layout, _ptr(dst), dst_layout, n_blocks,
                                             _stream(stream), err, _ERRLEN), err)


def kv_export_blocks(params, pool, blocks, n_blocks, out, stream=None):
    _calls.kv_export_blocks(params, pool, blocks, n_blocks, out, _stream(stream))


def kv_import_blocks(params, src, blocks, n_blocks, pool, stream=None):
    _calls.kv_import_blocks(params, src, blocks, n_blocks, pool, _stream(stream))


def attn_prep(params, X, qn_w, kn_w, pos, inv_freq, rope_sel, Q, Kb, Vb, row_table, pool, n_rows, stream=None):
    """All device tensors; rope_sel, row_table and pool may be None."""
    _calls.attn_prep(params, X, qn_w, kn_w, pos, inv_freq, rope_sel, Q, Kb, Vb, row_table, pool, n_rows, _stream(stream))


def decode_fused(pp, params, X, qn_w, kn_w, pos, inv_freq, rope_sel, row_table, pool, dp, O, stream=None):
    """attn_prep fused into the attention of a decode / short verify pass. dp: the DevicePass holding the records."""
    ws = dp.workspace
    _calls.attn_decode_fused(pp, params, X, qn_w, kn_w, pos, inv_freq, rope_sel, row_table, pool, dp.blocks, dp.desc, O, dp.tiles, dp.n_tiles,
                             dp.trees, dp.n_trees, dp.jobs, dp.n_jobs, dp.n_parts, dp.n_rows, ws, ws.nbytes, _stream(stream))


def head_gate(params, O, X, Wg, dots, n_rows, stream=None):
    """Device tensors. O (gated in place) or dots (fp32 [n_rows][H], written) may be None, not both."""
    _calls.head_gate(params, O, X, Wg, dots, n_rows, _stream(stream))


def chain_advance(trees, n_trees, pos, row_table, blocks, bt, ring=0, stream=None):
    """Device tensors: trees (TREE_DT bytes), pos / row_table int32 [rows][4], blocks int32."""
    _calls.chain_advance(trees, n_trees, pos, row_table, blocks, bt, ring, _stream(stream))


class DevicePass:
    """One planned pass resident on the device: uploads the records once and
    replays esp_attn_forward (what a decode chain does between host syncs)."""

    def __init__(self, params, trees, tiles, jobs, n_parts, n_rows, blocks, desc=None, pos=None, device="cuda",
                 pool_blocks=None, static=False, fused=False, rows_in_pool=False):
        """pool_blocks: blocks in the pool; when given, the records are checked on the host before the upload
        (fused: with the checks of a pass meant for decode_fused).
        static: run over the library's own scratch array (esp_attn_forward_static) instead of a workspace."""
        if pool_blocks is not None:
            validate(params, tiles, trees, jobs, n_parts, n_rows, blocks, pool_blocks, fused=fused, rows_in_pool=rows_in_pool)
        self.params = params
        self.static = static
        self.n_trees, self.n_tiles, self.n_jobs = len(trees), len(tiles), len(jobs)
        self.n_parts, self.n_rows = n_parts, n_rows
        self.trees_host, self.tiles_host, self.jobs_host = trees, tiles, jobs
        self.trees = to_dev(np.ascontiguousarray(trees, dtype=abi.TREE_DT), device)
        self.tiles = to_dev(np.ascontiguousarray(tiles, dtype=abi.TILE_DT), device)
        self.jobs = to_dev(np.ascontiguousarray(jobs, dtype=abi.COMBINE_DT), device) if len(jobs) else None
        self.blocks = to_dev(np.ascontiguousarray(blocks, dtype=np.int32), device) if blocks is not None else None
        self.desc = to_dev(np.ascontiguousarray(desc, dtype=np.int32), device) if desc is not None else None
        self.pos = to_dev(np.ascontiguousarray(pos, dtype=np.int32), device) if pos is not None else None
        nbytes = workspace_bytes(params, n_rows, n_parts)
        self.workspace = None if static else torch.empty(nbytes, dtype=torch.uint8, device=device)

    def run(self, Q, Kb, Vb, pool, O, stream=None, merge=True):
        """Enqueues the pass."""
        jobs, n_jobs = (self.jobs, self.n_jobs) if merge else (None, 0)
        if self.static:
            _calls.attn_forward_static(self.params, Q, Kb, Vb, pool, self.blocks, self.desc, self.pos, O, self.tiles, self.n_tiles, self.trees,
                                       self.n_trees, jobs, n_jobs, self.n_parts, self.n_rows, _stream(stream))
        else:
            ws = self.workspace
            _calls.attn_forward(self.params, Q, Kb, Vb, pool, self.blocks, self.desc, self.pos, O, self.tiles, self.n_tiles, self.trees,
                                self.n_trees, jobs, n_jobs, self.n_parts, self.n_rows, ws, ws.nbytes, _stream(stream))

    def merge(self, O, stream=None):
        if self.n_jobs:
            combine(self.params, O, self.jobs, self.n_jobs, self.n_parts, self.n_rows, self.workspace, stream)


def diff_params(weight, norm_w, eps, factor):
    """weight fp32 [H / 2], norm_w fp32 [2 * head_dim] or None: device tensors, kept alive by the record."""
    d = abi.DiffParams(_ptr(weight), _ptr(norm_w), eps, factor)
    d._keep = (weight, norm_w)
    return d


def attn_diff_rows(params, rows):
    """rows_per_tile to plan a pass of differential attention with whose trees have at most `rows` rows."""
    r = abi.attn_lib().esp_attn_diff_rows(C.byref(params), rows)
    if r <= 0:
        raise abi.EspError("parameters or rows that esp_attn_diff does not serve")
    return r


def attn_diff_hint(params, device=0):
    """(workgroups resident at once, workgroups per tile) of the differential attention kernel serving `params`."""
    err = C.create_string_buffer(_ERRLEN)
    n, g = C.c_int32(0), C.c_int32(0)
    abi.check(abi.attn_lib().esp_attn_diff_hint(C.byref(params), device, C.byref(n), C.byref(g), err, _ERRLEN), err)
    return n.value, abi.PlanGroups(g.value, params, diff=True)


class DiffPass:
    """One planned pass of differential attention resident on the device (the rows of the pass are in the pool when it runs)."""

    def __init__(self, params, diff, trees, tiles, jobs, n_parts, n_rows, blocks, device="cuda", pool_blocks=None):
        """pool_blocks: blocks in the pool; when given, the records are checked on the host before the upload. params stays the caller's
        record, read by every run; passes of another rows_per_tile need one of their own."""
        if pool_blocks is not None:
            validate(params, tiles, trees, jobs, n_parts, n_rows, blocks, pool_blocks, diff=True)
        self.params, self.diff, self.rows_per_tile = params, diff, params.rows_per_tile
        self.n_trees, self.n_tiles, self.n_jobs = len(trees), len(tiles), len(jobs)
        self.n_parts, self.n_rows = n_parts, n_rows
        self.trees = to_dev(np.ascontiguousarray(trees, dtype=abi.TREE_DT), device)
        self.tiles = to_dev(np.ascontiguousarray(tiles, dtype=abi.TILE_DT), device)
        self.jobs = to_dev(np.ascontiguousarray(jobs, dtype=abi.COMBINE_DT), device) if len(jobs) else None
        self.blocks = to_dev(np.ascontiguousarray(blocks, dtype=np.int32), device) if blocks is not None else None
        nbytes = abi.attn_lib().esp_attn_diff_workspace_bytes(C.byref(params), n_parts)
        self.workspace = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)

    def run(self, Q, pool, O, stream=None):
        if self.params.rows_per_tile != self.rows_per_tile:
            raise abi.EspError(f"rows_per_tile {self.params.rows_per_tile}: this pass was planned with {self.rows_per_tile} (one record for each)")
        ws = self.workspace
        _calls.attn_diff(self.params, self.diff, Q, pool, self.blocks, O, self.tiles, self.n_tiles, self.trees, self.n_trees, self.jobs, self.n_jobs,
                         self.n_parts, self.n_rows, ws, ws.nbytes, _stream(stream))


def shape_params(cap=0.0, slopes=None):
    """slopes fp32 [H] or None: a device tensor, kept alive by the record."""
    s = abi.ShapeParams(_ptr(slopes), None, cap, 0)
    s._keep = slopes
    return s


def attn_shaped_rows(params, rows):
    """rows_per_tile to plan a pass of attention with shaped scores with whose trees have at most `rows` rows."""
    r = abi.attn_lib().esp_attn_shaped_rows(C.byref(params), rows)
    if r <= 0:
        raise abi.EspError("parameters or rows that esp_attn_shaped does not serve")
    return r


def attn_shaped_hint(params, device=0):
    """(workgroups resident at once, workgroups per tile) of the kernel of attention with shaped scores serving `params`."""
    err = C.create_string_buffer(_ERRLEN)
    n, g = C.c_int32(0), C.c_int32(0)
    abi.check(abi.attn_lib().esp_attn_shaped_hint(C.byref(params), device, C.byref(n), C.byref(g), err, _ERRLEN), err)
    return n.value, abi.PlanGroups(g.value, params, shaped=True)


class ShapedPass:
    """One planned pass of attention with shaped scores resident on the device (the rows of the pass are in the pool when it runs)."""

    def __init__(self, params, shape, trees, tiles, jobs, n_parts, n_rows, blocks, spans=None, device="cuda", pool_blocks=None):
        """spans: int32 [n_rows][2], what each row sees (first key of its document, end of what is seen whichever way round), or None. The pass
        keeps copies of the records, with the spans that it was given. pool_blocks: blocks in the pool; when given, the records
        are checked on the host before the upload."""
        if pool_blocks is not None:
            validate(params, tiles, trees, jobs, n_parts, n_rows, blocks, pool_blocks, shaped=True)
        self.params, self.shape = abi.AttnParams.from_buffer_copy(params), abi.ShapeParams.from_buffer_copy(shape)
        self._keep = getattr(shape, "_keep", None)
        self.spans = None
        if spans is not None:
            spans = np.ascontiguousarray(spans, dtype=np.int32)
            if spans.shape != (n_rows, 2):
                raise abi.EspError(f"spans of shape {spans.shape}, {n_rows} rows of 2 expected")
            self.spans = to_dev(spans, device)
        self.shape.spans = _ptr(self.spans)
        self.n_trees, self.n_tiles, self.n_jobs = len(trees), len(tiles), len(jobs)
        self.n_parts, self.n_rows = n_parts, n_rows
        self.trees = to_dev(np.ascontiguousarray(trees, dtype=abi.TREE_DT), device)
        self.tiles = to_dev(np.ascontiguousarray(tiles, dtype=abi.TILE_DT), device)
        self.jobs = to_dev(np.ascontiguousarray(jobs, dtype=abi.COMBINE_DT), device) if len(jobs) else None
        self.blocks = to_dev(np.ascontiguousarray(blocks, dtype=np.int32), device) if blocks is not None else None
        nbytes = abi.attn_lib().esp_attn_shaped_workspace_bytes(C.byref(self.params), n_parts)
        self.workspace = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)

    def run(self, Q, pool, O, stream=None):
        ws = self.workspace
        _calls.attn_shaped(self.params, self.shape, Q, pool, self.blocks, O, self.tiles, self.n_tiles, self.trees, self.n_trees, self.jobs, self.n_jobs,
                           self.n_parts, self.n_rows, ws, ws.nbytes, _stream(stream))


def lowrank_params(D, rank, slices, dtype, x_ld, y_ld, n_adapters):
    """slices: (first column, columns) of each part of the projection that the adapters add to."""
    if not 1 <= len(slices) <= abi.ESP_LOWRANK_SLICES:
        raise abi.EspError(f"{len(slices)} slices (1 to {abi.ESP_LOWRANK_SLICES})")
    p = abi.LowRankParams(D, rank, len(slices), dtype, x_ld, y_ld, n_adapters, 0)
    for i, (off, width) in enumerate(slices):
        p.y_off[i], p.width[i] = off, width
    return p


def validate_lowrank(params, order, tiles, n_rows):
    """Host-side bounds check of a pass's records (numpy arrays) that the caller made or kept. Raises EspError. What
    host.plan_lowrank returns for n_rows rows passes."""
    order, tiles = np.ascontiguousarray(order, dtype=np.int32), np.ascontiguousarray(tiles, dtype=abi.LOWRANK_TILE_DT)
    err = C.create_string_buffer(_ERRLEN)
    abi.check(abi.attn_lib().esp_lowrank_validate(C.byref(params), order.ctypes.data, len(order), tiles.ctypes.data, len(tiles), n_rows, err, _ERRLEN),
              err)


class LowRankPass:
    """Which rows of a pass take which adapter, planned and resident on the device."""

    def __init__(self, params, adapter, device="cuda"):
        """adapter: int32 per row, -1 for a row without one. params: a layer's record may serve any number of passes. Each keeps a copy,
        with the rows_per_tile that its own tiles were planned with."""
        lib = abi.attn_lib()
        n_rows = len(adapter)
        params = abi.LowRankParams.from_buffer_copy(params)
        params.rows_per_tile = lib.esp_lowrank_rows(C.byref(params), max(n_rows, 1))
        if params.rows_per_tile <= 0:
            raise abi.EspError("parameters that esp_lowrank_add does not serve")
        self.params = params
        order, tiles = host.plan_lowrank(params, adapter)
        self.n_slots, self.n_tiles = len(order), len(tiles)
        self.order = to_dev(order, device) if self.n_slots else None
        self.tiles = to_dev(tiles, device) if self.n_tiles else None
        nbytes = lib.esp_lowrank_workspace_bytes(C.byref(params), self.n_tiles, self.n_slots)
        self.workspace = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)

    def run(self, X, A, B, scale, Y, stream=None):
        """Y += the adapters' products, in place."""
        ws = self.workspace
        _calls.lowrank_add(self.params, X, A, B, scale, Y, self.order, self.n_slots, self.tiles, self.n_tiles, ws, ws.nbytes, _stream(stream))


def logits_params(vocab, dtype, n_slots, n_masks=0, n_bias=0, in_ld=None, out_ld=None):
    return abi.LogitsParams(vocab, dtype, in_ld or vocab, out_ld or vocab, n_slots, n_masks, n_bias, 0)


class LogitsPass:
    """The records of the rows of a decode batch, resident on the device."""

    def __init__(self, params, rows, bias_tokens=None, device="cuda"):
        """rows: LOGITS_ROW_DT. bias_tokens: the host's copy of the bias entries' tokens; when given, records and entries are checked
        before the upload."""
        rows = np.ascontiguousarray(rows, dtype=abi.LOGITS_ROW_DT)
        lib = abi.attn_lib()
        if bias_tokens is not None:
            bias_tokens = np.ascontiguousarray(bias_tokens, dtype=np.int32)
            if len(bias_tokens) < params.n_bias:
                raise abi.EspError(f"{len(bias_tokens)} bias entries, {params.n_bias} named")
            err = C.create_string_buffer(_ERRLEN)
            abi.check(lib.esp_logits_validate(C.byref(params), rows.ctypes.data, len(rows), bias_tokens.ctypes.data, err, _ERRLEN), err)
        self.params, self.n_rows = params, len(rows)
        self.rows = to_dev(rows, device) if len(rows) else None
        nbytes = lib.esp_logits_workspace_bytes(C.byref(params), self.n_rows)
        self.workspace = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)

    def run(self, logits, out, tokens, bias_tokens, bias_values, masks, seen, counts, record=False, stream=None):
        """Device tensors; out or tokens may be None, and so may the arrays of which params counts 0 (histories, masks, bias entries).
        record: the tokens join their slots' histories."""
        ws = self.workspace
        _calls.logits_process(self.params, logits, out, tokens, self.rows, self.n_rows, bias_tokens, bias_values, masks, seen, counts, int(record), ws,
                              ws.nbytes, _stream(stream))


def history_record(params, seen, counts, tokens, slots, n, given, stream=None):
    _calls.history_record(params, seen, counts, tokens, slots, n, int(given), _stream(stream))


def history_clear(params, seen, counts, slots, n, stream=None):
    _calls.history_clear(params, seen, counts, slots, n, _stream(stream))


def linear_params(H, Hk, dk, dv, dtype, scale, n_states, row_decay=False, q_ld=None, k_ld=None, v_ld=None, o_ld=None, decay_ld=None):
    """row_decay: log decays [n_rows][H] (rows decay_ld apart) instead of [H]. Strides in elements, of rows without gaps by default."""
    return abi.LinearParams(H, Hk, dk, dv, dtype, q_ld or Hk * dk, k_ld or Hk * dk, v_ld or H * dv, o_ld or H * dv,
                            (decay_ld or H) if row_decay else 0, n_states, scale)


def validate_linear(params, tiles, n_few, n_parts, n_rows):
    """Host-side bounds check of a pass's records (numpy array) that the caller made or kept. Raises EspError. What
    host.plan_linear returns for n_rows rows passes."""
    tiles = np.ascontiguousarray(tiles, dtype=abi.LINEAR_TILE_DT)
    err = C.create_string_buffer(_ERRLEN)
    abi.check(abi.attn_lib().esp_linear_validate(C.byref(params), tiles.ctypes.data, len(tiles), n_few, n_parts, n_rows, err, _ERRLEN), err)


def linear_hint(params, device=0):
    """Workgroups of linear attention's chunked kernel that the device holds at once: what a pass is planned for."""
    err = C.create_string_buffer(_ERRLEN)
    n = C.c_int32(0)
    abi.check(abi.attn_lib().esp_linear_hint(C.byref(params), device, C.byref(n), err, _ERRLEN), err)
    return n.value


class LinearPass:
    """The sequences of a pass of linear attention, planned and resident on the device."""

    def __init__(self, params, seqs, n_rows, workgroups=None, device="cuda"):
        """seqs: LINEAR_SEQ_DT. params: a layer's record may serve any number of passes; each keeps a copy."""
        self.params, self.n_rows = abi.LinearParams.from_buffer_copy(params), n_rows
        if workgroups is None:
            workgroups = linear_hint(params, torch.device(device).index or 0)
        tiles, self.n_few, self.n_parts = host.plan_linear(params, seqs, n_rows, workgroups)
        self.n_tiles = len(tiles)
        self.tiles = to_dev(tiles, device) if self.n_tiles else None
        nbytes = abi.attn_lib().esp_linear_workspace_bytes(C.byref(params), self.n_parts)
        self.workspace = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)

    def run(self, Q, K, V, decay, states, O, stream=None):
        """Device tensors; Q, K, V may be slices of one projection's rows (their strides in params). states are updated in place."""
        ws = self.workspace
        _calls.linear_attn(self.params, Q, K, V, decay, states, O, self.tiles, self.n_tiles, self.n_few, self.n_parts, self.n_rows, ws, ws.nbytes,
                           _stream(stream))
