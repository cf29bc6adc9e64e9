"""Prompt prefill of a ragged batch through the routed experts on the tcgen05
tensor cores (the LFM2-24B-A2B-shaped configuration).

Per layer: post-attention and routing of every prompt row (`yn_rows_route`,
bit-identical to the single-row path); the rows' fp16 K-permuted copy
(`yn_gather_f16_kperm`, in pair order); the grouping of the (row, column) pairs by expert, as
the reference's prefill sweep plans its staging groups (sweep.py:80-138); the grouped gate/up + SwiGLU and down GEMMs
(`yn_tc_experts`, 128 weight rows x up to 256 rows per tile); the combine in
column order plus the residual (`yn_pairs_combine`). The grouping runs on the
device (`yn_prefill_plan`, by a rule `yn_prefill_plan_by_rule`); `plan_prefill` is its host restatement.

Two things can be chosen: `rule` routes by a `routing.RouteRule` instead of the
softmax top-k (the logits of `yn_rows_route` through `yn_route_scored`), and
`experts="int8"` holds the routed experts as 8-bit matrices with channel scales
(made once from the records) and runs a layer's experts as `int8.int8_experts`.
"""
from __future__ import annotations

import ctypes as C
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _lib
from .device import DeviceLayer, ExpertArena, dims_struct, fill_synthetic_experts, stream_ptr
from .formats import RecordSpec
from .int8 import Int8Matrix, int8_experts, quantize_rows
from .routing import RouteRule, check_choice_bias, route_scored
from .synthetic import StackConfig, dense_layer

TILE_ROWS = 256      # token rows per tile
UP_UNITS = 64        # gate/up units per tile (128 weight rows)
DOWN_ROWS = 128      # down output rows per tile


def route_logits(ws: torch.Tensor, dims: _lib.Dims, rows: int) -> torch.Tensor:
    """The router logits (rows, E) fp32 that `yn_rows_route` of that many rows left in its workspace."""
    p = C.c_void_p()
    _lib.check(_lib.lib().yn_rows_route_logits(C.byref(dims), rows, ws.data_ptr(), C.byref(p)))
    off, n = p.value - ws.data_ptr(), rows * dims.n_experts * 4
    return ws[off:off + n].view(torch.float32).view(rows, dims.n_experts)


class TcTile(C.Structure):
    _fields_ = [("e", C.c_int32), ("p0", C.c_int32), ("n", C.c_int32), ("u0", C.c_int32)]


def plan_prefill(ids: np.ndarray, n_experts: int, inter: int, hidden: int):
    """Pairs grouped by expert (ascending id, rows in order inside an expert).
    Returns pair_row (P,), pair_of (T, K), gate/up tiles and down tiles as
    int32 arrays of (e, p0, n, u0)."""
    ids = np.asarray(ids)
    T, K = ids.shape
    flat = ids.reshape(-1)
    order = np.argsort(flat, kind="stable")          # pair p -> flat index t * K + j
    pair_row = (order // K).astype(np.int32)
    pair_of = np.empty(T * K, np.int32)
    pair_of[order] = np.arange(T * K, dtype=np.int32)
    experts, starts, counts = np.unique(flat[order], return_index=True, return_counts=True)
    up, down = [], []
    for e, p0, n in zip(experts.tolist(), starts.tolist(), counts.tolist()):
        for c0 in range(0, n, TILE_ROWS):
            m = min(TILE_ROWS, n - c0)
            up += [(e, p0 + c0, m, u) for u in range(0, inter, UP_UNITS)]
            down += [(e, p0 + c0, m, r) for r in range(0, hidden, DOWN_ROWS)]
    return (pair_row, pair_of.reshape(T, K), np.array(up, np.int32).reshape(-1, 4),
            np.array(down, np.int32).reshape(-1, 4))


def int8_matrices(arena: ExpertArena, spec: RecordSpec, n_experts: int, hidden: int, inter: int,
                  first_slot: int = 0) -> Tuple[Int8Matrix, Int8Matrix, Int8Matrix]:
    """The gate, up and down matrices (E, I, H), (E, I, H), (E, H, I) of the records in
    slots first_slot.. of an arena, dequantised and quantised again with one scale per
    output channel. Once, at load time."""
    lib, out = _lib.lib(), []
    dev = arena.buf.device
    with torch.cuda.device(dev):
        for part, (rows, cols) in enumerate(((inter, hidden), (inter, hidden), (hidden, inter))):
            codes = torch.zeros((n_experts, rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=dev)
            scales = torch.empty((n_experts, rows), dtype=torch.float32, device=dev)
            full = torch.empty((rows, cols), dtype=torch.float32, device=dev)
            for e in range(n_experts):
                rec = arena.base + (first_slot + e) * arena.slot_bytes
                m = _lib.QMat(*(rec + spec.offsets[3 * part + i] for i in range(3)), rows, cols, spec.bits,
                              spec.group_size)
                _lib.check(lib.yn_dequantize(C.byref(m), full.data_ptr(), stream_ptr()))
                q = quantize_rows(full)
                codes[e, :, :cols] = q.codes
                scales[e] = q.scales
            out.append(Int8Matrix(codes[..., :cols], scales))
    return tuple(out)


class PrefillStack:
    """Resident experts and dense weights of `layers` of `cfg`, and the
    buffers for prompts of up to `max_rows` rows in total. A layer runs
    entirely on the device (routing, grouping, GEMMs, combine): no host
    synchronisation. A layer's output is the residual and the routed experts: a shared
    expert is not in it (the backend's prompt pass has one), and ``experts="int8"`` refuses a
    configuration that has one. rule / choice_bias: route by a rule, with a bias fp32 on its choice,
    (len(layers), E): row i is that of ``layers[i]``. experts: "records" (4-bit codes as they are) or "int8"."""

    def __init__(self, cfg: StackConfig, max_rows: int, device: str = "cuda",
                 layers: Optional[Sequence[int]] = None, rule: Optional[RouteRule] = None,
                 choice_bias: Optional[torch.Tensor] = None, experts: str = "records"):
        if experts not in ("records", "int8"):
            raise ValueError(f"experts must be 'records' or 'int8', not {experts!r}")
        if experts == "int8" and cfg.shared_inter:
            raise NotImplementedError("experts='int8' runs the routed experts only: the configuration has a shared one")
        if rule is not None and rule.top_k != cfg.top_k:
            raise ValueError(f"the rule chooses {rule.top_k} experts, the configuration {cfg.top_k}")
        self.cfg = cfg
        self.layer_ids = list(range(cfg.n_layers)) if layers is None else list(layers)
        check_choice_bias(choice_bias, rule, len(self.layer_ids), cfg.n_experts)
        self.rule, self.choice_bias = rule, choice_bias
        self.int8: Optional[List[Tuple[Int8Matrix, Int8Matrix, Int8Matrix]]] = [] if experts == "int8" else None
        self.device = torch.device(device)
        self.dims = dims_struct(cfg)
        self.arenas: List[ExpertArena] = []
        self.layers: List[DeviceLayer] = []
        for l in self.layer_ids:
            spec = cfg.record_spec(l)
            arena = ExpertArena(cfg.n_experts, spec.slot_bytes, self.device)
            fill_synthetic_experts(arena, cfg, l)
            if self.int8 is not None:
                self.int8.append(int8_matrices(arena, spec, cfg.n_experts, cfg.hidden, cfg.moe_inter))
                arena = ExpertArena(1, 16, self.device)      # the records are not kept
            self.arenas.append(arena)
            self.layers.append(DeviceLayer(cfg, l, dense_layer(cfg, l), arena, 0, None, self.device))
        self.structs = [L.struct() for L in self.layers]
        lib = _lib.lib()
        H, K, I = cfg.hidden, cfg.top_k, cfg.moe_inter
        T, P = max_rows, max_rows * K
        dev = self.device
        self.max_rows = max_rows
        nb = int(lib.yn_rows_route_bytes(C.byref(self.dims), max_rows))
        if not nb:
            raise ValueError("max_rows outside what the routing workspace supports")
        self.route_ws = torch.zeros(nb, dtype=torch.uint8, device=dev)
        mu, md = C.c_int32(0), C.c_int32(0)
        _lib.check(lib.yn_prefill_max_tiles(C.byref(self.dims), max_rows, C.byref(mu), C.byref(md)))
        self.max_up, self.max_dn = mu.value, md.value
        self.n_tiles = torch.zeros(2, dtype=torch.int32, device=dev)
        self.pair_row = torch.empty(P, dtype=torch.int32, device=dev)
        self.pair_of = torch.empty(P, dtype=torch.int32, device=dev)
        self.x = torch.empty((T, H), dtype=torch.bfloat16, device=dev)
        self.ids = torch.empty((T, K), dtype=torch.int32, device=dev)
        self.w = torch.empty((T, K), dtype=torch.float32, device=dev)
        self.tiles_up = self.tiles_dn = self.x16 = self.act = self.y = None
        if self.int8 is None:      # what the record experts need; int8_experts takes a workspace of its own
            self.tiles_up = torch.empty((self.max_up, 4), dtype=torch.int32, device=dev)
            self.tiles_dn = torch.empty((self.max_dn, 4), dtype=torch.int32, device=dev)
            self.x16 = torch.empty((P, H), dtype=torch.float16, device=dev)  # rows in pair order
            self.act = torch.empty((P, I), dtype=torch.bfloat16, device=dev)
            self.y = torch.empty((P, H), dtype=torch.bfloat16, device=dev)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)
        self.ping = torch.empty((2, T, H), dtype=torch.bfloat16, device=dev)

    def layer(self, i: int, h: torch.Tensor, out: torch.Tensor, stream=None, gemm_events=None) -> None:
        """Layer i (index into `layer_ids`) of T = h.shape[0] rows. gemm_events:
        optional list that receives (start, end) CUDA events around the two
        grouped GEMM launches (of the records; the 8-bit experts are one call)."""
        lib, cfg = _lib.lib(), self.cfg
        T, H = h.shape[0], cfg.hidden
        if T > self.max_rows:
            raise ValueError("more rows than the buffers hold")
        if self.int8 is not None and gemm_events is not None:
            raise ValueError("gemm_events: the 8-bit experts have no events between their kernels")
        st = stream_ptr(stream)
        D, L = C.byref(self.dims), C.byref(self.structs[i])
        _lib.check(lib.yn_rows_route(D, L, h.data_ptr(), T, self.x.data_ptr(), self.ids.data_ptr(), self.w.data_ptr(),
                                     self.route_ws.data_ptr(), self.route_ws.numel(), st))
        if self.rule is not None:
            route_scored(route_logits(self.route_ws, self.dims, T), self.rule,
                         None if self.choice_bias is None else self.choice_bias[i], stream=stream,
                         out=(self.ids[:T], self.w[:T]))
        if self.int8 is not None:
            int8_experts(self.x[:T], self.ids[:T], self.w[:T], *self.int8[i], residual=h, stream=stream, out=out,
                         err=self.err)
            return
        plan = lib.yn_prefill_plan if self.rule is None else lib.yn_prefill_plan_by_rule
        _lib.check(plan(D, self.ids.data_ptr(), T, self.pair_row.data_ptr(), self.pair_of.data_ptr(),
                        self.tiles_up.data_ptr(), self.max_up, self.tiles_dn.data_ptr(), self.max_dn,
                        self.n_tiles.data_ptr(), self.err.data_ptr(), st))
        P = T * cfg.top_k
        _lib.check(lib.yn_gather_f16_kperm(self.x.data_ptr(), self.pair_row.data_ptr(), P, H, self.x16.data_ptr(), st))
        if gemm_events is not None:
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record(stream)
        nt = self.n_tiles.data_ptr()
        _lib.check(lib.yn_tc_experts(D, L, 0, self.tiles_up.data_ptr(), self.max_up, nt, self.x16.data_ptr(), P,
                                     self.act.data_ptr(), None, self.err.data_ptr(), st))
        _lib.check(lib.yn_tc_experts(D, L, 1, self.tiles_dn.data_ptr(), self.max_dn, nt + 4, self.act.data_ptr(), P,
                                     None, self.y.data_ptr(), self.err.data_ptr(), st))
        if gemm_events is not None:
            e1.record(stream)
            gemm_events.append((e0, e1))
        _lib.check(lib.yn_pairs_combine(D, self.y.data_ptr(), self.pair_of.data_ptr(), self.w.data_ptr(), None,
                                        h.data_ptr(), T, out.data_ptr(), st))

    def plan(self, T: int):
        """Host copies of the last layer's ids, pair -> row and (row, column) -> pair (record experts)."""
        if self.int8 is not None:
            raise ValueError("the 8-bit experts keep their grouping to themselves")
        K = self.cfg.top_k
        return (self.ids[:T].cpu().numpy(), self.pair_row[:T * K].cpu().numpy(),
                self.pair_of[:T * K].cpu().numpy().reshape(T, K))

    def prefill(self, h: torch.Tensor, stream=None, gemm_events=None) -> torch.Tensor:
        """Every layer for the rows h (T, H) bf16; returns the last layer's output."""
        T = h.shape[0]
        self.ping[0, :T].copy_(h)
        for i in range(len(self.layer_ids)):
            self.layer(i, self.ping[i % 2, :T], self.ping[(i + 1) % 2, :T], stream, gemm_events)
        return self.ping[len(self.layer_ids) % 2, :T]

    def check_error(self) -> int:
        torch.cuda.synchronize(self.device)
        code = int(self.err.item())
        rc = C.c_int32(0)
        _lib.check(_lib.lib().yn_route_error(self.route_ws.data_ptr(), C.byref(self.dims), stream_ptr(),
                                             C.byref(rc)))
        self.err.zero_()
        return code or rc.value


def kperm_inverse(a: np.ndarray) -> np.ndarray:
    """Natural column order of a K-permuted (…, cols) array."""
    cols = a.shape[-1]
    k = np.arange(cols)
    p = k & 7
    pos = (k & ~7) | np.where(p < 4, 2 * p, 2 * (p - 4) + 1)
    return a[..., pos]
