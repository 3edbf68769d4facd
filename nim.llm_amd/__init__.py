"""MI355X token sampler -- Python host mirror of nimllm's `Sampler` over the C ABI.

The compute lives in ``libnimllm_sampler.so`` (HIP kernels for gfx950, built from
``csrc/`` by ``csrc/Makefile``); this module only marshals arguments through
ctypes.  It mirrors src/nimllm/sampler.nim:

* ``SamplerParams`` (:11-21), ``defaultSampling`` (:28-31), ``greedySampling`` (:33-35)
* ``newSampler`` / ``Sampler.accept`` / ``Sampler.sample`` (:37-43, :59-121) for one
  row, and ``BatchSampler`` for B independent rows on the device.

Beside the sampler stand the output projection (``lm_head``) and what a layer
does between projections for contexts that decode together: rotary positions
(``rope_plan``, ``rope``), the paged cache (``PagedCache``, ``cache_*``) and the
attention over it (``paged_attention``).

There is no CPU fallback: without the built library or a GPU every entry
point raises.
"""
from __future__ import annotations

import ctypes
import functools
import math
import os
from dataclasses import dataclass, field
from typing import NamedTuple, Optional, Sequence

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libnimllm_sampler.so")

NLS_OK = 0
PATH_GREEDY, PATH_TOPK, PATH_FULL, PATH_GENERIC = 1, 2, 3, 4
# accept entries that append nothing (a row that ended this step):
# NLS_ACCEPT_SKIP for host int64 ids, NLS_ACCEPT_SKIP32 for device int32 ids
ACCEPT_SKIP = -(1 << 63)
ACCEPT_SKIP32 = -(1 << 31)

EXPORTED = (
    "nls_default_sampling", "nls_greedy_sampling", "nls_create", "nls_destroy",
    "nls_set_stream", "nls_batch", "nls_vocab", "nls_accept", "nls_accept_row",
    "nls_accept_device", "nls_generate_step", "nls_clear_history", "nls_sample", "nls_sample_host",
    "nls_sample_host_noalloc",
    "nls_synchronize", "nls_rng_uniforms", "nls_get_rng_state", "nls_set_rng_state",
    "nls_top_tokens", "nls_row_nll", "nls_softmax_rows", "nls_log_prob", "nls_expf_device",
    "nls_expf_forms_device",
    "nls_rows_workspace", "nls_top_tokens_ws", "nls_row_nll_ws", "nls_softmax_rows_ws", "nls_log_prob_ws",
    "nls_profile_next",
    "nls_profile_next_generic", "nls_get_plan", "nls_status_string", "nls_last_error",
    "nls_lm_head_workspace", "nls_lm_head", "nls_lm_head_row_bytes", "nls_argmax",
    "nls_rope_frequencies", "nls_rope", "nls_cache_append", "nls_paged_attention_workspace", "nls_paged_attention",
    "nls_cache_workspace", "nls_cache_reserve", "nls_cache_fork", "nls_cache_release", "nls_cache_compact",
    "nls_cache_copy_pages", "nls_cache_page_bytes", "nls_cache_read",
    "nls_cache_reorder_workspace", "nls_cache_reorder", "nls_beam_workspace", "nls_beam_select",
)


class NlsLora(ctypes.Structure):
    """nls_lora: a LoRA adapter on the output matrix (LoraPair, model.nim:34-39)."""

    _fields_ = [("d_a", ctypes.c_void_p), ("d_b", ctypes.c_void_p), ("rank", ctypes.c_int32),
                ("scale", ctypes.c_float)]


def _c_struct(doc, name, **fields):
    return type(name, (ctypes.Structure,), {"__doc__": doc, "_fields_": list(fields.items())})


_vp, _i32, _i64, _f64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_double
NlsHeads = _c_struct("nls_heads: rows of heads", "NlsHeads", d=_vp, token_stride=_i64, head_stride=_i64)
NlsRopeScaling = _c_struct("nls_rope_scaling", "NlsRopeScaling", kind=_i32, base=_f64, factor=_f64, original_context=_f64,
                           beta_fast=_f64, beta_slow=_f64, attn_factor=_f64, freq_factors=ctypes.POINTER(_f64))
NlsRopePlan = _c_struct("nls_rope_plan", "NlsRopePlan", d_freqs=_vp, dim=_i32, interleaved=_i32,
                        amplitude=ctypes.c_float)
NlsPagedKv = _c_struct("nls_paged_kv: one layer of the cache", "NlsPagedKv", d_kv=_vp, type=_i32, pages=_i32,
                       page_size=_i32, kv_heads=_i32, head_dim=_i32, page_stride=_i64, value_offset=_i64,
                       head_stride=_i64, token_stride=_i64, d_table=_vp, table_stride=_i64, slots=_i32, max_pages=_i32,
                       d_lens=_vp)
NlsChunks = _c_struct("nls_chunks: the new tokens of a call", "NlsChunks", seqs=_i32, tokens=_i32, d_starts=_vp,
                      d_slots=_vp)
NlsPagePool = _c_struct("nls_page_pool: the pages of all layers", "NlsPagePool", d_kv=_vp, layers=_i32,
                        page_bytes=_i64, layer_stride=_i64, page_stride=_i64)
NlsPageTables = _c_struct("nls_page_tables: who holds which page", "NlsPageTables", d_table=_vp, table_stride=_i64,
                          slots=_i32, max_pages=_i32, d_lens=_vp, d_refs=_vp, pages=_i32, page_size=_i32)


class NlsParams(ctypes.Structure):
    _fields_ = [
        ("temperature", ctypes.c_double),
        ("top_k", ctypes.c_int64),
        ("top_p", ctypes.c_double),
        ("min_p", ctypes.c_double),
        ("repeat_penalty", ctypes.c_double),
        ("repeat_last_n", ctypes.c_int64),
        ("presence_penalty", ctypes.c_double),
        ("frequency_penalty", ctypes.c_double),
        ("seed", ctypes.c_int64),
        ("logit_bias_ids", ctypes.POINTER(ctypes.c_int64)),
        ("logit_bias_values", ctypes.POINTER(ctypes.c_double)),
        ("logit_bias_count", ctypes.c_int64),
    ]


class NlsDebug(ctypes.Structure):
    _fields_ = [
        ("n", ctypes.c_void_p),
        ("ncand", ctypes.c_void_p),
        ("cand_ids", ctypes.c_void_p),
        ("cand_probs", ctypes.c_void_p),
        ("total", ctypes.c_void_p),
        ("path", ctypes.c_void_p),
        ("cap", ctypes.c_int32),
    ]


class NlsPlan(ctypes.Structure):
    _fields_ = [
        ("stream_threads", ctypes.c_int32),
        ("slices", ctypes.c_int32),
        ("generic_launch", ctypes.c_int32),
        ("streamed_rows", ctypes.c_int32),
        ("first_unit_bytes", ctypes.c_int64),
        ("k64", ctypes.c_int32),
        ("walk_split", ctypes.c_int32),
        ("floor_slices", ctypes.c_int32),
    ]


class SamplerError(RuntimeError):
    pass


_lib = None


def lib():
    """Load the HIP library (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise SamplerError(f"{LIB_PATH} is missing: build it with `make -C {HERE}/csrc`")
        L = ctypes.CDLL(LIB_PATH)
        P = ctypes.POINTER
        vp = ctypes.c_void_p
        L.nls_default_sampling.restype = NlsParams
        L.nls_greedy_sampling.restype = NlsParams
        L.nls_create.argtypes = [P(NlsParams), ctypes.c_int32, ctypes.c_int64, vp, P(vp)]
        L.nls_destroy.argtypes = [vp]
        L.nls_set_stream.argtypes = [vp, vp]
        L.nls_batch.argtypes = [vp]
        L.nls_batch.restype = ctypes.c_int32
        L.nls_vocab.argtypes = [vp]
        L.nls_vocab.restype = ctypes.c_int64
        L.nls_accept.argtypes = [vp, P(ctypes.c_int64), ctypes.c_int32]
        L.nls_accept_row.argtypes = [vp, ctypes.c_int32, P(ctypes.c_int64), ctypes.c_int32]
        L.nls_accept_device.argtypes = [vp, vp]
        L.nls_generate_step.argtypes = [vp, vp, vp, vp, vp, ctypes.c_int32, vp]
        L.nls_clear_history.argtypes = [vp]
        L.nls_sample.argtypes = [vp, vp, vp, vp, P(NlsDebug)]
        L.nls_sample_host.argtypes = [vp, P(ctypes.c_float), P(ctypes.c_int64)]
        L.nls_sample_host_noalloc.argtypes = [vp, P(ctypes.c_float), P(ctypes.c_int64)]
        L.nls_synchronize.argtypes = [vp]
        L.nls_rng_uniforms.argtypes = [ctypes.c_int64, ctypes.c_int64, P(ctypes.c_double)]
        L.nls_get_rng_state.argtypes = [vp, ctypes.c_int32, P(ctypes.c_uint64), P(ctypes.c_uint64)]
        L.nls_set_rng_state.argtypes = [vp, ctypes.c_int32, ctypes.c_uint64, ctypes.c_uint64]
        L.nls_top_tokens.argtypes = [vp, ctypes.c_int32, ctypes.c_int64, ctypes.c_int32, vp, vp, vp]
        L.nls_row_nll.argtypes = [vp, ctypes.c_int32, ctypes.c_int64, vp, vp, vp]
        L.nls_softmax_rows.argtypes = [vp, ctypes.c_int32, ctypes.c_int64, vp, vp]
        L.nls_log_prob.argtypes = [vp, ctypes.c_int32, ctypes.c_int64, vp, vp, vp, vp]
        L.nls_rows_workspace.argtypes = [ctypes.c_int32, ctypes.c_int32, ctypes.c_int64, ctypes.c_int32]
        L.nls_rows_workspace.restype = ctypes.c_size_t
        ws = [vp, ctypes.c_size_t, vp]  # the workspace, its bytes, the stream
        L.nls_top_tokens_ws.argtypes = L.nls_top_tokens.argtypes[:-1] + ws
        L.nls_row_nll_ws.argtypes = L.nls_row_nll.argtypes[:-1] + ws
        L.nls_softmax_rows_ws.argtypes = L.nls_softmax_rows.argtypes[:-1] + ws
        L.nls_log_prob_ws.argtypes = L.nls_log_prob.argtypes[:-1] + ws
        L.nls_expf_device.argtypes = [vp, vp, ctypes.c_int64, vp]
        L.nls_expf_forms_device.argtypes = L.nls_expf_device.argtypes
        L.nls_profile_next.argtypes = [vp, vp, vp]
        L.nls_profile_next_generic.argtypes = [vp, vp, vp]
        L.nls_get_plan.argtypes = [vp, P(NlsPlan), P(ctypes.c_int32)]
        L.nls_status_string.argtypes = [ctypes.c_int]
        L.nls_status_string.restype = ctypes.c_char_p
        L.nls_last_error.restype = ctypes.c_char_p
        L.nls_lm_head_workspace.argtypes = [ctypes.c_int32, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32,
                                            ctypes.c_int32]
        L.nls_lm_head_workspace.restype = ctypes.c_size_t
        L.nls_lm_head_row_bytes.argtypes = [ctypes.c_int32, ctypes.c_int64]
        L.nls_lm_head_row_bytes.restype = ctypes.c_int64
        L.nls_argmax.argtypes = [vp, ctypes.c_int32, ctypes.c_int64, vp, vp]
        L.nls_lm_head.argtypes = [vp, ctypes.c_int32, ctypes.c_int64, ctypes.c_int64, vp, ctypes.c_int32, vp,
                                  ctypes.c_int32, P(NlsLora), vp, ctypes.c_size_t, vp]
        L.nls_lm_head.restype = ctypes.c_int32
        i32, i64, hp, kp, cp = ctypes.c_int32, ctypes.c_int64, P(NlsHeads), P(NlsPagedKv), P(NlsChunks)
        L.nls_rope_frequencies.argtypes = [P(NlsRopeScaling), i32, P(ctypes.c_double), P(ctypes.c_double)]
        L.nls_rope.argtypes = [P(NlsRopePlan), i32, hp, hp, i32, i32, i32, vp, i32, vp]
        L.nls_cache_append.argtypes = [kp, cp, P(NlsRopePlan), i32, hp, hp, i32, hp, hp, vp]
        L.nls_paged_attention_workspace.argtypes = [kp, cp, i32, i32, i64, i32]
        L.nls_paged_attention_workspace.restype = ctypes.c_size_t
        L.nls_paged_attention.argtypes = [kp, cp, i32, hp, hp, i32, ctypes.c_float, i32, vp, vp, i32, i64] + ws
        pp, tp = P(NlsPagePool), P(NlsPageTables)
        L.nls_cache_page_bytes.argtypes = [i32, i32, i32, i32]
        L.nls_cache_page_bytes.restype = i64
        L.nls_cache_read.argtypes = [kp, cp, i32, hp, hp, vp]
        L.nls_cache_workspace.argtypes = [tp, i32]
        L.nls_cache_workspace.restype = ctypes.c_size_t
        L.nls_cache_reserve.argtypes = [tp, vp, vp] + ws
        L.nls_cache_fork.argtypes = [pp, tp, vp, vp, i32, vp] + ws
        L.nls_cache_release.argtypes = [tp, vp, i32, vp] + ws
        L.nls_cache_compact.argtypes = [pp, tp, vp] + ws
        L.nls_cache_reorder_workspace.argtypes = [tp]
        L.nls_cache_reorder_workspace.restype = ctypes.c_size_t
        L.nls_cache_reorder.argtypes = [pp, tp, vp, vp] + ws
        L.nls_beam_workspace.argtypes = [i32, i32, i64]
        L.nls_beam_workspace.restype = ctypes.c_size_t
        L.nls_beam_select.argtypes = [vp, i32, i32, i64, vp, vp, vp, i32, vp, vp, vp, vp] + ws
        L.nls_cache_copy_pages.argtypes = [pp, i32, vp, vp, i32, vp]
        _lib = L
    return _lib


def check(status: int, what: str = "") -> None:
    if status != NLS_OK:
        L = lib()
        raise SamplerError(f"{what}: {L.nls_status_string(status).decode()} "
                           f"({L.nls_last_error().decode()})")


@dataclass
class SamplerParams:
    """SamplerParams (sampler.nim:11-21).  Omitted fields are zero, as in Nim."""

    temperature: float = 0.0
    topK: int = 0
    topP: float = 0.0
    minP: float = 0.0
    repeatPenalty: float = 0.0
    repeatLastN: int = 0
    presencePenalty: float = 0.0
    frequencyPenalty: float = 0.0
    seed: int = 0
    logitBias: dict = field(default_factory=dict)


def defaultSampling() -> SamplerParams:
    """sampler.nim:28-31"""
    return SamplerParams(temperature=0.7, topK=40, topP=0.95, minP=0.05,
                         repeatPenalty=1.1, repeatLastN=64, seed=-1)


def greedySampling() -> SamplerParams:
    """sampler.nim:33-35"""
    return SamplerParams(temperature=0.0, topK=0, topP=1.0, repeatPenalty=1.0, seed=0)


def _to_c(p: SamplerParams, keep: list) -> NlsParams:
    c = NlsParams()
    c.temperature = p.temperature
    c.top_k = p.topK
    c.top_p = p.topP
    c.min_p = p.minP
    c.repeat_penalty = p.repeatPenalty
    c.repeat_last_n = p.repeatLastN
    c.presence_penalty = p.presencePenalty
    c.frequency_penalty = p.frequencyPenalty
    c.seed = p.seed
    n = len(p.logitBias)
    if n:
        ids = (ctypes.c_int64 * n)(*[int(k) for k in p.logitBias.keys()])
        vals = (ctypes.c_double * n)(*[float(v) for v in p.logitBias.values()])
        keep.extend([ids, vals])
        c.logit_bias_ids = ids
        c.logit_bias_values = vals
    c.logit_bias_count = n
    return c


def rng_uniforms(seed: int, n: int):
    """The first n values of rand(1.0) after initRand(seed) (Nim std/random)."""
    arr = (ctypes.c_double * max(n, 1))()
    check(lib().nls_rng_uniforms(seed, n, arr), "nls_rng_uniforms")
    return [arr[i] for i in range(n)]


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


class BatchSampler:
    """B independent samplers (one per row) on the current HIP device.

    ``sample`` takes a device tensor of shape [B, V] (float32) and returns the
    sampled ids as a device int32 tensor; it is asynchronous on ``stream``.
    """

    def __init__(self, params: Sequence[SamplerParams], vocab: int, stream=None):
        import torch

        self._torch = torch
        L = lib()
        keep: list = []
        B = len(params)
        arr = (NlsParams * B)(*[_to_c(p, keep) for p in params])
        self._stream = stream
        self.B, self.V = B, int(vocab)
        h = ctypes.c_void_p()
        check(L.nls_create(arr, B, int(vocab), self._stream_ptr(), ctypes.byref(h)), "nls_create")
        self._h = h

    def _stream_ptr(self):
        s = self._stream
        if s is None:
            return None
        return ctypes.c_void_p(s.cuda_stream if hasattr(s, "cuda_stream") else int(s))

    def close(self):
        if getattr(self, "_h", None):
            lib().nls_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def accept(self, ids, row: Optional[int] = None):
        """accept (sampler.nim:41-43): one id per row ([B]) or [B, n] ids; or
        ids for a single `row`.  ACCEPT_SKIP entries append nothing."""
        import numpy as np

        a = np.ascontiguousarray(np.asarray(ids, dtype=np.int64))
        L = lib()
        if row is not None:
            a = a.reshape(-1)
            check(L.nls_accept_row(self._h, int(row), a.ctypes.data_as(ctypes.POINTER(ctypes.c_int64)),
                                   a.size), "nls_accept_row")
            return
        a = a.reshape(self.B, -1)
        check(L.nls_accept(self._h, a.ctypes.data_as(ctypes.POINTER(ctypes.c_int64)), a.shape[1]),
              "nls_accept")

    def accept_device(self, d_ids):
        """One id per row from device int32 [B]; ACCEPT_SKIP32 appends nothing."""
        assert d_ids.dtype == self._torch.int32 and d_ids.is_cuda and d_ids.numel() == self.B
        check(lib().nls_accept_device(self._h, ctypes.c_void_p(d_ids.data_ptr())), "nls_accept_device")

    def clear_history(self):
        check(lib().nls_clear_history(self._h), "nls_clear_history")

    def sample(self, logits, u=None, out=None, debug_cap: int = 0):
        """sample (sampler.nim:59-121) for every row.  `u` (float64 [B], device)
        stands for each row's rand(1.0); None draws from the rows' own RNGs.
        With debug_cap > 0 returns (ids, debug dict of device tensors)."""
        torch = self._torch
        assert logits.is_cuda and logits.dtype == torch.float32 and logits.is_contiguous()
        assert tuple(logits.shape) == (self.B, self.V), (logits.shape, self.B, self.V)
        if u is not None:
            assert u.is_cuda and u.dtype == torch.float64 and u.numel() == self.B and u.is_contiguous()
        if out is None:
            out = torch.empty(self.B, dtype=torch.int32, device=logits.device)
        dbgp = None
        dbg = None
        if debug_cap > 0:
            dev = logits.device
            dbg = {
                "n": torch.full((self.B,), -1, dtype=torch.int32, device=dev),
                "ncand": torch.full((self.B,), -1, dtype=torch.int32, device=dev),
                "cand_ids": torch.full((self.B, debug_cap), -1, dtype=torch.int32, device=dev),
                "cand_probs": torch.zeros((self.B, debug_cap), dtype=torch.float32, device=dev),
                "total": torch.zeros((self.B,), dtype=torch.float32, device=dev),
                "path": torch.zeros((self.B,), dtype=torch.int32, device=dev),
            }
            dbgp = NlsDebug(dbg["n"].data_ptr(), dbg["ncand"].data_ptr(), dbg["cand_ids"].data_ptr(),
                            dbg["cand_probs"].data_ptr(), dbg["total"].data_ptr(),
                            dbg["path"].data_ptr(), debug_cap)
        check(lib().nls_sample(self._h, ctypes.c_void_p(logits.data_ptr()),
                               ctypes.c_void_p(_ptr(u)) if u is not None else None,
                               ctypes.c_void_p(out.data_ptr()),
                               ctypes.byref(dbgp) if dbgp is not None else None), "nls_sample")
        return (out, dbg) if debug_cap > 0 else out

    def generate_step(self, logits, eog, done, u=None, out=None):
        """One step of batched generation (chat.nim:204-208 for every row): rows
        with done == 0 sample; a row drawing an id in `eog` (int32 device
        tensor) gets done = 1 and accepts nothing, the others accept their id.
        Finished rows sample nothing (out = -1) and keep their RNG state.
        `done`: int32 device tensor [B], zero before the first step.  Returns out."""
        torch = self._torch
        assert logits.is_cuda and logits.dtype == torch.float32 and logits.is_contiguous()
        assert tuple(logits.shape) == (self.B, self.V)
        assert done.is_cuda and done.dtype == torch.int32 and done.numel() == self.B and done.is_contiguous()
        assert eog.is_cuda and eog.dtype == torch.int32 and eog.is_contiguous()
        if u is not None:
            assert u.is_cuda and u.dtype == torch.float64 and u.numel() == self.B and u.is_contiguous()
        if out is None:
            out = torch.empty(self.B, dtype=torch.int32, device=logits.device)
        check(lib().nls_generate_step(self._h, ctypes.c_void_p(logits.data_ptr()),
                                      ctypes.c_void_p(_ptr(u)) if u is not None else None,
                                      ctypes.c_void_p(out.data_ptr()),
                                      ctypes.c_void_p(eog.data_ptr()) if eog.numel() else None,
                                      int(eog.numel()), ctypes.c_void_p(done.data_ptr())),
              "nls_generate_step")
        return out

    def sample_host(self, logits):
        """Blocking: host [B, V] float32 logits -> host int64 [B] ids."""
        import numpy as np

        x = np.ascontiguousarray(np.asarray(logits, dtype=np.float32).reshape(self.B, self.V))
        o = np.zeros(self.B, dtype=np.int64)
        check(lib().nls_sample_host(self._h, x.ctypes.data_as(ctypes.POINTER(ctypes.c_float)),
                                    o.ctypes.data_as(ctypes.POINTER(ctypes.c_int64))), "nls_sample_host")
        return o

    def sample_host_noalloc(self, logits):
        """sample_host through the library's static staging (nothing allocated)."""
        import numpy as np

        x = np.ascontiguousarray(np.asarray(logits, dtype=np.float32).reshape(self.B, self.V))
        o = np.zeros(self.B, dtype=np.int64)
        check(lib().nls_sample_host_noalloc(self._h, x.ctypes.data_as(ctypes.POINTER(ctypes.c_float)),
                                            o.ctypes.data_as(ctypes.POINTER(ctypes.c_int64))),
              "nls_sample_host_noalloc")
        return o

    def profile_next(self, start_event, stop_event):
        """Time the next sample()'s streaming kernel with two torch.cuda.Events
        (recorded on this sampler's stream)."""
        check(lib().nls_profile_next(self._h, ctypes.c_void_p(start_event.cuda_event),
                                     ctypes.c_void_p(stop_event.cuda_event)), "nls_profile_next")

    def profile_next_generic(self, start_event, stop_event):
        """Time the next sample()'s whole-row kernel (when it launches one)."""
        check(lib().nls_profile_next_generic(self._h, ctypes.c_void_p(start_event.cuda_event),
                                             ctypes.c_void_p(stop_event.cuda_event)), "nls_profile_next_generic")

    def plan(self):
        """(NlsPlan, per-row list: 1 where the streaming kernel runs the row)."""
        p = NlsPlan()
        rows = (ctypes.c_int32 * self.B)()
        check(lib().nls_get_plan(self._h, ctypes.byref(p), rows), "nls_get_plan")
        return p, list(rows)

    def synchronize(self):
        check(lib().nls_synchronize(self._h), "nls_synchronize")

    def rng_state(self, row: int):
        a0, a1 = ctypes.c_uint64(), ctypes.c_uint64()
        check(lib().nls_get_rng_state(self._h, row, ctypes.byref(a0), ctypes.byref(a1)), "rng")
        return a0.value, a1.value

    def set_rng_state(self, row: int, a0: int, a1: int):
        check(lib().nls_set_rng_state(self._h, row, a0, a1), "rng")


class Sampler:
    """One nimllm Sampler (sampler.nim:23-26) backed by a one-row BatchSampler.

    ``sample(logits)`` accepts a host sequence/ndarray (through
    nls_sample_host: the kernel reads it from the handle's pinned staging) or a
    1-D device tensor, and returns the id as a Python int.
    """

    def __init__(self, p: SamplerParams, vocab: int):
        self.params = p
        self._b = BatchSampler([p], vocab)

    def accept(self, tok: int):
        self._b.accept([int(tok)])

    def sample(self, logitsIn) -> int:
        torch = self._b._torch
        if isinstance(logitsIn, torch.Tensor) and logitsIn.is_cuda:
            out = self._b.sample(logitsIn.reshape(1, -1).contiguous().float())
            return int(out.cpu()[0])
        return int(self._b.sample_host(logitsIn)[0])


def newSampler(p: Optional[SamplerParams] = None, vocab: int = 0) -> Sampler:
    """newSampler (sampler.nim:37-39).  The vocabulary size is fixed per sampler
    here because the device buffers are sized from it."""
    if vocab <= 0:
        raise SamplerError("newSampler needs the vocabulary size")
    return Sampler(p if p is not None else defaultSampling(), vocab)


TOP_TOKENS_MAX = 2048  # largest number of entries per row nls_top_tokens returns


# nls_rows_workspace's calls
_ROWS_SOFTMAX, _ROWS_LOG_PROB, _ROWS_TOP_TOKENS, _ROWS_NLL = range(4)
# Rows shorter than this want none (nls_rows_workspace answers 0): a short call
# is bound by its launch, and the question would cost it a tenth (row_nll of
# 8 x 8000: 8.6 us without it, 9.4 with).
_ROWS_WORK_FROM = {_ROWS_SOFTMAX: 8192, _ROWS_LOG_PROB: 8192, _ROWS_TOP_TOKENS: 8192, _ROWS_NLL: 40960}


def _rows_work(op: int, x, rows: int, V: int, n: int = 0):
    """The workspace of a call over the rows of x (None where it wants none, or
    where the memory has no room for it: topTokens' is half the logits' size for
    short rows), from torch's allocator on the current stream, and its bytes."""
    if V < _ROWS_WORK_FROM[op]:
        return None, 0
    import torch

    need = int(lib().nls_rows_workspace(op, rows, V, n))
    if not need:
        return None, 0
    try:
        return torch.empty(need, dtype=torch.uint8, device=x.device), need
    except torch.OutOfMemoryError:  # the calls run without one too
        return None, 0


def top_tokens_device(logits, n: int = 5):
    """topTokens (sampler.nim:123-130) for a [rows, V] float32 device tensor:
    returns int32 ids and float32 probabilities, both [rows, min(n, V)], in the
    reference's order (probability descending, ascending id on ties)."""
    import torch

    x = logits if logits.dim() == 2 else logits.reshape(1, -1)
    assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
    rows, V = x.shape
    m = max(0, min(n, V))
    ids = torch.empty((rows, max(n, 1)), dtype=torch.int32, device=x.device)
    probs = torch.empty((rows, max(n, 1)), dtype=torch.float32, device=x.device)
    stream = torch.cuda.current_stream(x.device).cuda_stream
    work, wb = _rows_work(_ROWS_TOP_TOKENS, x, rows, V, n)
    check(lib().nls_top_tokens_ws(ctypes.c_void_p(x.data_ptr()), rows, V, n,
                                  ctypes.c_void_p(ids.data_ptr()), ctypes.c_void_p(probs.data_ptr()),
                                  _ptr(work), wb, ctypes.c_void_p(stream)), "nls_top_tokens")
    return ids[:, :m], probs[:, :m]


def topTokens(logits, n: int = 5):
    """topTokens (sampler.nim:123-130): the n most probable ids of one row of
    logits (any float32 sequence or tensor) with their probabilities, as a list
    of (id, probability) pairs, computed on the device."""
    import numpy as np
    import torch

    x = logits if torch.is_tensor(logits) else torch.from_numpy(np.ascontiguousarray(logits, dtype=np.float32))
    x = x.reshape(1, -1).to(device="cuda", dtype=torch.float32).contiguous()
    ids, probs = top_tokens_device(x, n)
    return [(int(i), float(p)) for i, p in zip(ids[0].tolist(), probs[0].tolist())]


def argmax_device(logits):
    """argmax (sampler.nim:45-49) of every row of a [rows, V] (or [V])
    float32 device tensor: int32 [rows], the first index of each row's
    greatest value (a NaN never taken; a NaN at index 0 answers 0)."""
    import torch

    x = logits if logits.dim() == 2 else logits.reshape(1, -1)
    assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
    rows, V = x.shape
    out = torch.empty(rows, dtype=torch.int32, device=x.device)
    stream = torch.cuda.current_stream(x.device).cuda_stream
    check(lib().nls_argmax(ctypes.c_void_p(x.data_ptr()) if V else None, rows, V,
                           ctypes.c_void_p(out.data_ptr()), ctypes.c_void_p(stream)), "nls_argmax")
    return out


def argmax(logits) -> int:
    """argmax (sampler.nim:45-49) of one row of logits (any float32 sequence
    or tensor), computed on the device."""
    import numpy as np
    import torch

    x = logits if torch.is_tensor(logits) else torch.from_numpy(np.ascontiguousarray(logits, dtype=np.float32))
    x = x.reshape(1, -1).to(device="cuda", dtype=torch.float32).contiguous()
    return int(argmax_device(x)[0].item())


def row_nll_device(logits, targets):
    """perplexity's per-position term (src/nimllm/model.nim:578-583) for a
    [rows, V] float32 device tensor and int32 target ids [rows]: float64
    -(l[t] - max) + ln(sum of exp(l - max)) per row."""
    import torch

    x = logits if logits.dim() == 2 else logits.reshape(1, -1)
    assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
    t = targets.to(device=x.device, dtype=torch.int32).contiguous()
    rows, V = x.shape
    assert t.numel() == rows
    out = torch.empty(rows, dtype=torch.float64, device=x.device)
    stream = torch.cuda.current_stream(x.device).cuda_stream
    work, wb = _rows_work(_ROWS_NLL, x, rows, V)
    check(lib().nls_row_nll_ws(ctypes.c_void_p(x.data_ptr()), rows, V, ctypes.c_void_p(t.data_ptr()),
                               ctypes.c_void_p(out.data_ptr()), _ptr(work), wb, ctypes.c_void_p(stream)),
          "nls_row_nll")
    return out


def softmax_device(logits, out=None):
    """softmaxInPlace (src/nimllm/sampler.nim:51-57) of every row of a
    [rows, V] (or [V]) float32 device tensor; `out` may be `logits` itself
    (the reference's in-place form).  Returns out."""
    import torch

    x = logits if logits.dim() == 2 else logits.reshape(1, -1)
    assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
    rows, V = x.shape
    if out is None:
        out = torch.empty_like(logits)
    assert out.is_cuda and out.dtype == torch.float32 and out.is_contiguous() and out.numel() == x.numel()
    stream = torch.cuda.current_stream(x.device).cuda_stream
    work, wb = _rows_work(_ROWS_SOFTMAX, x, rows, V)
    check(lib().nls_softmax_rows_ws(ctypes.c_void_p(x.data_ptr()), rows, V, ctypes.c_void_p(out.data_ptr()),
                                    _ptr(work), wb, ctypes.c_void_p(stream)), "nls_softmax_rows")
    return out


def log_prob_device(logits, targets):
    """logProb's per-token term (nimllm-doc-en.md:1700-1707) for a [rows, V]
    float32 device tensor and int32 target ids [rows]: (p[target] float32,
    ln(float64(p[target])) float64) per row, p = softmaxInPlace of the row."""
    import torch

    x = logits if logits.dim() == 2 else logits.reshape(1, -1)
    assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
    t = targets.to(device=x.device, dtype=torch.int32).contiguous()
    rows, V = x.shape
    assert t.numel() == rows
    prob = torch.empty(rows, dtype=torch.float32, device=x.device)
    logp = torch.empty(rows, dtype=torch.float64, device=x.device)
    stream = torch.cuda.current_stream(x.device).cuda_stream
    work, wb = _rows_work(_ROWS_LOG_PROB, x, rows, V)
    check(lib().nls_log_prob_ws(ctypes.c_void_p(x.data_ptr()), rows, V, ctypes.c_void_p(t.data_ptr()),
                                ctypes.c_void_p(prob.data_ptr()), ctypes.c_void_p(logp.data_ptr()),
                                _ptr(work), wb, ctypes.c_void_p(stream)), "nls_log_prob")
    return prob, logp


def log_prob(context_logits, continuation):
    """logProb (nimllm-doc-en.md:1700-1707) given the logits the model
    produced before each continuation token ([len, V] device tensor) and the
    continuation's ids: the float64 sum of ln(p[id]) in token order."""
    _, lp = log_prob_device(context_logits, continuation)
    total = 0.0
    for v in lp.cpu().tolist():
        total += v
    return total


def perplexity(logits, targets):
    """exp of the mean per-position term over the rows (model.nim:570-589,
    for logits already evaluated), computed on the device."""
    import math

    nll = row_nll_device(logits, targets)
    return math.exp(float(nll.sum().item()) / max(1, nll.numel()))


def expf_device(x, out=None):
    """Correctly rounded exp of a float32 device tensor."""
    import torch

    assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
    if out is None:
        out = torch.empty_like(x)
    check(lib().nls_expf_device(ctypes.c_void_p(x.data_ptr()), ctypes.c_void_p(out.data_ptr()),
                                x.numel(), None), "nls_expf_device")
    return out


def inf_bias() -> float:
    return -math.inf


# GGML type codes (src/nimllm/quant.nim:14-19) nls_lm_head reads
GGML_TYPES = {"F32": 0, "F16": 1, "Q4_0": 2, "Q4_1": 3, "Q5_0": 6, "Q5_1": 7, "Q8_0": 8, "Q2_K": 10,
              "Q3_K": 11, "Q4_K": 12, "Q5_K": 13, "Q6_K": 14, "Q8_K": 15, "BF16": 30}


def lm_head_workspace(ggml_type: int, cols: int, nb: int, lora_rank: int = 0, exact: bool = False) -> int:
    return int(lib().nls_lm_head_workspace(ggml_type, cols, nb, lora_rank, int(exact)))


def lm_head(weight, ggml_type: int, rows: int, cols: int, x, exact: bool = False, lora=None, out=None,
            work=None):
    """matmul(m.output, x, y, nb) (src/nimllm/model.nim:179-200) on the device:
    weight is a uint8 device tensor of rows * rowBytes(type, cols) GGUF bytes,
    x a float32 device tensor [nb, cols] (or [cols]); returns y [nb, rows]
    float32 ([rows] for a 1-D x).  exact is the reference's exactMatmul;
    lora = (a [rank, cols], b [rows, rank], scale) device tensors.  `work`
    may pass a preallocated uint8 device workspace."""
    import torch

    x2 = x if x.dim() == 2 else x.reshape(1, -1)
    assert x2.is_cuda and x2.dtype == torch.float32 and x2.is_contiguous() and x2.shape[1] == cols
    rb = int(lib().nls_lm_head_row_bytes(ggml_type, cols))
    if rb < 0:
        raise SamplerError(f"lm_head: type {ggml_type} with cols={cols} is not a readable GGUF row "
                           "(rowBytes raises)")
    assert weight.is_cuda and weight.is_contiguous() and weight.dtype == torch.uint8
    assert weight.device == x2.device, "lm_head: weight and x on different devices"
    assert weight.numel() >= rows * rb, (
        f"lm_head: weight holds {weight.numel()} bytes, rows x rowBytes = {rows * rb}")
    nb = x2.shape[0]
    if out is None:
        out = torch.empty((nb, rows), dtype=torch.float32, device=x2.device)
    assert out.is_cuda and out.dtype == torch.float32 and out.is_contiguous() and out.numel() == nb * rows
    lo = None
    rank = 0
    if lora is not None:
        a, b, scale = lora
        assert a.is_contiguous() and b.is_contiguous() and a.dtype == torch.float32 and b.dtype == torch.float32
        assert a.is_cuda and b.is_cuda and a.device == x2.device and b.device == x2.device
        assert a.dim() == 2 and b.dim() == 2
        rank = a.shape[0]
        assert tuple(a.shape) == (rank, cols) and tuple(b.shape) == (rows, rank), (
            f"lm_head: LoRA a {tuple(a.shape)} must be ({rank}, {cols}), b {tuple(b.shape)} ({rows}, {rank})")
        lo = NlsLora(a.data_ptr(), b.data_ptr(), rank, float(scale))
    need = lm_head_workspace(ggml_type, cols, nb, rank, exact)
    if work is None or work.numel() < need:
        work = torch.empty(max(need, 1), dtype=torch.uint8, device=x2.device)
    stream = torch.cuda.current_stream(x2.device).cuda_stream
    check(lib().nls_lm_head(ctypes.c_void_p(weight.data_ptr()), ggml_type, rows, cols,
                            ctypes.c_void_p(x2.data_ptr()), nb, ctypes.c_void_p(out.data_ptr()), int(exact),
                            ctypes.byref(lo) if lo is not None else None, ctypes.c_void_p(work.data_ptr()),
                            work.numel(), ctypes.c_void_p(stream)), "nls_lm_head")
    return out if x.dim() == 2 else out.reshape(rows)


# ---------------------------------------------------------------- attention over a paged cache


_ELEM_TYPES: dict = {}


def _elem_type(t) -> int:
    code = _ELEM_TYPES.get(t.dtype)
    if code is None:
        import torch

        _ELEM_TYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 30})
        code = _ELEM_TYPES.get(t.dtype)
        if code is None:
            raise SamplerError(f"element type {t.dtype} is not float32, float16 or bfloat16")
    return code


# The checks below are raised, not asserted: the C ABI sees addresses alone, and
# what is wrong in lengths, types or devices would be read on the GPU, under
# python -O too.


def _ints(device: int, t):
    """The address of a contiguous int32 tensor on the device (None: none)."""
    if t is None:
        return None
    if t.get_device() != device:
        raise AssertionError("tensors of one call on different devices")
    if not (t.element_size() == 4 and not t.is_floating_point() and t.is_contiguous()):
        raise AssertionError("int32 tensors, contiguous")
    return t.data_ptr()


def _heads(device: int, t, dtype):
    """A [tokens, heads, head_dim] tensor as nls_heads."""
    if not (t.get_device() == device and t.dtype == dtype):
        raise AssertionError("tensors of one call: one device, one element type")
    s = t.stride()
    if not (len(s) == 3 and (s[2] == 1 or t.shape[2] <= 1)):
        raise AssertionError("rows of heads: [tokens, heads, head_dim], elements side by side")
    return NlsHeads(t.data_ptr(), s[0], s[1])


def _launch(device: int, what: str, *args):
    """The call on the device's current stream, with that device current.  (The
    raw forms of torch.cuda.current_stream and current_device: 5 us less, of a
    call that takes 10.)"""
    import torch

    C = torch._C
    call = getattr(lib(), what)
    if C._cuda_getDevice() == device:
        status = call(*args, C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            status = call(*args, C._cuda_getCurrentRawStream(device))
    if status != NLS_OK:
        check(status, what)


@dataclass
class RopePlan:
    """Rotary positions of a model: each pair's angle per position (float64 device
    tensor [dim / 2]), whether pairs are neighbours (2j, 2j + 1) or halves
    (j, j + dim / 2), and the amplitude."""

    freqs: object
    interleaved: bool = True
    amplitude: float = 1.0

    def _c(self, device: int):
        f = self.freqs
        if not (f.get_device() == device and f.element_size() == 8 and f.is_floating_point() and f.dim() == 1 and
                f.is_contiguous()):
            raise AssertionError("rope plan: float64 [dim / 2] on the call's device")
        return NlsRopePlan(f.data_ptr(), 2 * f.numel(), self.interleaved, self.amplitude)


ROPE_SCALINGS = {"none": 0, "linear": 1, "yarn": 2}


def rope_frequencies(dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                     original_context: float = 0.0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                     attn_factor: float = 1.0, freq_factors=None):
    """(angles per position of the dim / 2 pairs, amplitude), on the host: the
    rope.* keys of a GGUF file and its rope_freqs tensor (freq_factors)."""
    if scaling not in ROPE_SCALINGS:
        raise SamplerError(f"rope scaling {scaling!r} is none of {sorted(ROPE_SCALINGS)}")
    n = max(dim // 2, 1)
    ff = None
    if freq_factors is not None:
        ff = [float(f) for f in freq_factors]
        if len(ff) != dim // 2:
            raise AssertionError(f"freq_factors: {len(ff)} entries, dim / 2 = {dim // 2}")
        ff = (ctypes.c_double * n)(*ff)
    out, amp = (ctypes.c_double * n)(), ctypes.c_double()
    s = NlsRopeScaling(ROPE_SCALINGS[scaling], base, factor, original_context, beta_fast, beta_slow, attn_factor, ff)
    check(lib().nls_rope_frequencies(ctypes.byref(s), dim, out, ctypes.byref(amp)), "nls_rope_frequencies")
    return list(out)[:dim // 2], amp.value


def rope_plan(dim: int, interleaved: bool = True, device="cuda", **scaling) -> RopePlan:
    """A RopePlan for the first `dim` elements of each head (rope_frequencies'
    arguments); interleaved as llama's GGUF files have it, halves as qwen's."""
    import torch

    freqs, amp = rope_frequencies(dim, **scaling)
    return RopePlan(torch.tensor(freqs, dtype=torch.float64, device=device), interleaved, amp)


def rope(x, positions, plan: RopePlan, inverse: bool = False, out=None):
    """x [tokens, heads, head_dim] with the first elements of each head turned by
    its token's position (int32 [tokens]); `inverse` takes a gradient back.
    `out` may be x.  Returns out."""
    dev, dt = x.get_device(), x.dtype
    if out is None:
        import torch

        out = torch.empty(x.shape, dtype=dt, device=x.device)
    tokens, heads, dim = x.shape
    if not (dev >= 0 and out.shape == x.shape and positions.numel() == tokens):
        raise AssertionError("rope: x on the GPU, out of its shape, a position per token")
    _launch(dev, "nls_rope", plan._c(dev), _elem_type(x), _heads(dev, x, dt), _heads(dev, out, dt), tokens, heads, dim,
            _ints(dev, positions), inverse)
    return out


@functools.lru_cache(maxsize=None)
def _format_of(kind: str, kv_heads: int, page_size: int, head_dim: int):
    """(type code, bytes of a page) of a PageFormat's sizes."""
    t = {"q8_0": 8, "q4_0": 2}.get(kind)
    if t is None:
        raise SamplerError(f"page format {kind!r} is neither q8_0 nor q4_0")
    n = -1
    if 0 < kv_heads < 1 << 31 and 0 < page_size <= 4096 and 0 < head_dim <= 256:
        n = int(lib().nls_cache_page_bytes(t, kv_heads, page_size, head_dim))
    if n < 0:
        raise SamplerError(f"page format {kind} of {kv_heads} heads of {head_dim}, {page_size} tokens: pages are of 16 to "
                           "4096 tokens (a power of two), heads of a multiple of 32 up to 256")
    return t, n


class PageFormat(NamedTuple):
    """Pages whose keys and values are blocks of 32 elements of a head, an fp16
    factor and a code of 8 or 4 bits each: kind "q8_0" or "q4_0", as GGUF's types
    of those names hold.  One layer of such a cache is a uint8 tensor [pages,
    page_bytes], whose pages are 16-byte aligned."""

    kind: str
    kv_heads: int
    page_size: int
    head_dim: int

    @property
    def type(self) -> int:
        return _format_of(*self)[0]

    @property
    def page_bytes(self) -> int:
        return _format_of(*self)[1]


def _kv_dims(kv, fmt):
    """(kv_heads, page_size, head_dim) of a layer."""
    return kv.shape[2:] if fmt is None else fmt[1:]


def _paged_kv(dev: int, kv, table, lens, fmt=None):
    st = kv.stride()
    if fmt is not None:
        kind, size = _format_of(*fmt)
        if not (dev >= 0 and len(st) == 2 and kv.element_size() == 1 and st[1] == 1 and kv.shape[1] == size):
            raise AssertionError("a layer of blocks on the GPU: uint8 [pages, page_bytes] of its format")
        pages, (_, kv_heads, page_size, dim) = kv.shape[0], fmt
        st = st[0], 0, 0, 0
    else:
        pages, two, kv_heads, page_size, dim = kv.shape
        if not (dev >= 0 and two == 2 and st[4] == 1):
            raise AssertionError("a layer of the cache on the GPU: [pages, 2, kv_heads, page_size, head_dim], elements side by side")
        kind = _elem_type(kv)
    slots, per = table.shape
    ts = table.stride()
    if not (table.get_device() == dev and table.dtype == lens.dtype and ts[1] == 1 and lens.numel() == slots):
        raise AssertionError("the page table: int32 [slots, pages], rows side by side")
    return NlsPagedKv(kv.data_ptr(), kind, pages, page_size, kv_heads, dim, st[0], st[1], st[2], st[3],
                      table.data_ptr(), ts[0], slots, per, _ints(dev, lens))


def _in_range(window: int, max_new: int, max_len: int):
    """Numbers that the C ABI takes whole: ctypes cuts others to 32 bits."""
    if not (0 <= window < 1 << 31 and 0 <= max_new < 1 << 31 and 0 <= max_len < 1 << 63):
        raise AssertionError("window and max_new: 0 .. 2^31 - 1, max_len: 0 .. 2^63 - 1")


def _chunks(dev: int, tokens: int, starts, slots):
    seqs = starts.numel() - 1
    if not (seqs >= 0 and (slots is None or slots.numel() == seqs)):
        raise AssertionError("starts [sequences + 1], slots [sequences]")
    return NlsChunks(seqs, tokens, _ints(dev, starts), _ints(dev, slots))


def cache_append(kv, table, lens, starts, k, v, q=None, plan: Optional[RopePlan] = None, slots=None, out=None,
                 fmt: Optional[PageFormat] = None):
    """The new tokens of a layer into the cache: k turned by `plan` (None: as it
    is) and v, both [tokens, kv_heads, head_dim], to the pages of their
    positions; q [tokens, heads, head_dim] turned into `out` (which may be q).
    Sequence i's tokens are rows starts[i] .. starts[i + 1] and the last ones of
    slot slots[i] (i when None), whose lens count them already.  fmt: the format
    of a cache of blocks.  Returns out."""
    dev, dt = kv.get_device(), k.dtype
    tokens, kv_heads, dim = k.shape
    of = _kv_dims(kv, fmt)
    if not (k.shape == v.shape and kv_heads == of[0] and dim == of[2]):
        raise AssertionError("k and v: [tokens, kv_heads, head_dim] of the cache's heads")
    heads, cq, co = 0, None, None
    if q is not None:
        if out is None:
            import torch

            out = torch.empty(q.shape, dtype=dt, device=q.device)
        heads = q.shape[1]
        if not (out.shape == q.shape and q.shape[0] == tokens and q.shape[2] == dim):
            raise AssertionError("q and out: [tokens, heads, head_dim] of k's tokens and head_dim")
        cq, co = _heads(dev, q, dt), _heads(dev, out, dt)
    else:
        if out is not None:
            raise AssertionError("out without q")
    _launch(dev, "nls_cache_append", _paged_kv(dev, kv, table, lens, fmt), _chunks(dev, tokens, starts, slots),
            None if plan is None else plan._c(dev), _elem_type(k), cq, co, heads, _heads(dev, k, dt), _heads(dev, v, dt))
    return out


def cache_read(kv, table, lens, starts, tokens: int, dtype=None, k=None, v=None, slots=None,
               fmt: Optional[PageFormat] = None):
    """The cached keys and values of the sequences' last tokens (cache_append's
    starts and slots) as rows again: (k, v), both [tokens, kv_heads, head_dim] of
    `dtype` (float32 by default, or that of a k and v given).  Rows without a
    place in the cache are 0, rows of no sequence are left as they were."""
    import torch

    dev, of = kv.get_device(), _kv_dims(kv, fmt)
    shape = (tokens, of[0], of[2])
    given = k if k is not None else v
    dt = dtype or (torch.float32 if given is None else given.dtype)
    if k is None:
        k = torch.empty(shape, dtype=dt, device=kv.device)
    if v is None:
        v = torch.empty(shape, dtype=dt, device=kv.device) if given is not None else torch.empty_like(k)
    if not (k.shape == shape and v.shape == shape):
        raise AssertionError("k and v: [tokens, kv_heads, head_dim] of the cache's heads")
    _launch(dev, "nls_cache_read", _paged_kv(dev, kv, table, lens, fmt), _chunks(dev, tokens, starts, slots), _elem_type(k),
            _heads(dev, k, dt), _heads(dev, v, dt))
    return k, v


def paged_attention(q, kv, table, lens, starts, max_new: int = 0, max_len: int = 0, scale: Optional[float] = None,
                    window: int = 0, first=None, slots=None, out=None, lse=None, work=None,
                    fmt: Optional[PageFormat] = None):
    """Attention of the new tokens' q [tokens, heads, head_dim] over their slots'
    cached keys and values (cache_append's arguments): causal, at most `window`
    keys back when that is > 0, from key first[slot] on when given.  scale:
    1 / sqrt(head_dim) by default.  max_new and max_len: what the caller knows of
    the longest chunk and context (0: nothing); they choose how the work is
    split, not what comes out.  lse: True, or a float32 [tokens, heads] tensor,
    for the logarithm of each row's sum.  Rows of no sequence keep what `out` and
    `lse` hold.  `work`: a preallocated uint8 workspace of
    paged_attention_workspace() bytes.  fmt: the format of a cache of blocks.
    Returns out, or (out, lse)."""
    import torch

    dev, dt = kv.get_device(), q.dtype
    tokens, heads, dim = q.shape
    _in_range(window, max_new, max_len)
    if out is None:
        out = torch.empty(q.shape, dtype=dt, device=q.device)
    if lse is False:
        lse = None
    elif lse is True:
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device)
    elif lse is not None:
        if not (lse.get_device() == dev and lse.dtype == torch.float32 and lse.is_contiguous() and
                lse.shape == (tokens, heads)):
            raise AssertionError("lse: float32 [tokens, heads], contiguous")
    if not (out.shape == q.shape and dim == _kv_dims(kv, fmt)[2] and (first is None or first.numel() == lens.numel())):
        raise AssertionError("out: q's shape; q: the cache's head_dim; first: a key per slot")
    c, ch = _paged_kv(dev, kv, table, lens, fmt), _chunks(dev, tokens, starts, slots)
    cq, co, cf = _heads(dev, q, dt), _heads(dev, out, dt), _ints(dev, first)
    need = lib().nls_paged_attention_workspace(c, ch, heads, max_new, max_len, window)
    if need and (work is None or work.numel() < need):
        work = torch.empty(need, dtype=torch.uint8, device=q.device)
    elif work is not None:
        if not (work.get_device() == dev and work.dtype == torch.uint8 and work.is_contiguous()):
            raise AssertionError("work: uint8, contiguous, on the call's device")
    _launch(dev, "nls_paged_attention", c, ch, _elem_type(q), cq, co, heads, dim ** -0.5 if scale is None else scale,
            window, cf, None if lse is None else lse.data_ptr(), max_new, max_len, _ptr(work), need)
    return out if lse is None else (out, lse)


def paged_attention_workspace(q, kv, table, lens, starts, max_new: int = 0, max_len: int = 0, window: int = 0,
                              fmt: Optional[PageFormat] = None) -> int:
    """Bytes of the workspace paged_attention takes for these arguments, for a
    caller that keeps one (each call in flight needs its own)."""
    _in_range(window, max_new, max_len)
    return int(lib().nls_paged_attention_workspace(_paged_kv(kv.get_device(), kv, table, lens, fmt),
                                                   _chunks(kv.get_device(), q.shape[0], starts, None), q.shape[1], max_new,
                                                   max_len, window))


PAGES_DONE, PAGES_NONE_LEFT, PAGES_ROW_FULL, PAGES_BAD_ENTRY = range(4)


def _page_pool(dev: int, kv, fmt=None):
    st, n = kv.stride(), kv.element_size()
    if fmt is not None:
        if not (kv.get_device() == dev and kv.dim() == 3 and n == 1 and st[2] == 1 and kv.shape[2] == fmt.page_bytes):
            raise AssertionError("a cache of blocks: uint8 [layers, pages, page_bytes] of its format")
        return NlsPagePool(kv.data_ptr(), kv.shape[0], kv.shape[2], st[0], st[1])
    layers, _, two, heads, page_size, dim = kv.shape
    dense = 1  # elements of a page so far, in the order of the strides
    for stride, size in sorted(zip(st[2:], kv.shape[2:])):
        if size != 1:
            dense = dense * size if stride == dense else 0
    if not (kv.get_device() == dev and two == 2 and dense == 2 * heads * page_size * dim):
        raise AssertionError("the cache: [layers, pages, 2, kv_heads, page_size, head_dim], each page's contents side by side")
    return NlsPagePool(kv.data_ptr(), layers, dense * n, st[0] * n, st[1] * n)


def _page_size(kv, fmt) -> int:
    return kv.shape[4] if fmt is None else fmt.page_size


def _page_tables(dev: int, table, lens, refs, page_size: int):
    slots, per = table.shape
    ts = table.stride()
    if not 0 < page_size <= 4096:
        raise AssertionError("page_size: a power of two up to 4096")
    if not (dev >= 0 and table.get_device() == dev and table.dtype == refs.dtype and ts[1] == 1 and
            (lens is None or lens.numel() == slots)):
        raise AssertionError("the page table: int32 [slots, pages], rows side by side")
    return NlsPageTables(table.data_ptr(), ts[0], slots, per, _ints(dev, lens), _ints(dev, refs), refs.numel(), page_size)


def _pages_call(dev: int, what: str, refs, need: int, *args):
    """One of the page calls with its workspace of `need` bytes; returns its int32
    word."""
    import torch

    # the word, then the workspace from the next 256 bytes on
    both = torch.empty(need // 4 + 64, dtype=torch.int32, device=refs.device)
    at = both.data_ptr()
    _launch(dev, what, *args, at, at + 256, need)
    return both[:1]


def cache_reserve(table, lens, refs, page_size: int, counts):
    """Slot s grows by counts[s] (int32) tokens: the lowest free pages, in the
    slots' order, and lens += counts.  Returns the status word (PAGES_DONE, or
    why nothing was done) as an int32 device tensor [1]."""
    dev = refs.get_device()
    if counts.numel() != table.shape[0]:
        raise AssertionError("counts: one per slot")
    t = _page_tables(dev, table, lens, refs, page_size)
    return _pages_call(dev, "nls_cache_reserve", refs, lib().nls_cache_workspace(t, 0), t, _ints(dev, counts))


def cache_fork(kv, table, lens, refs, src, dst, fmt: Optional[PageFormat] = None):
    """The empty slots dst[i] (int32) become copies of the slots src[i]: full
    pages shared, the last partial page copied in every layer of kv (fmt: the
    format of a cache of blocks, uint8 [layers, pages, page_bytes]).  Returns the
    status word."""
    dev, n = refs.get_device(), src.numel()
    if not (n == dst.numel() and kv.shape[1] == refs.numel()):
        raise AssertionError("src and dst of one length; refs: one per page of kv")
    t = _page_tables(dev, table, lens, refs, _page_size(kv, fmt))
    return _pages_call(dev, "nls_cache_fork", refs, lib().nls_cache_workspace(t, n), _page_pool(dev, kv, fmt), t, _ints(dev, src), _ints(dev, dst), n)


def cache_release(table, lens, refs, slots, page_size: int):
    """The slots (int32) let go of their pages and are empty.  Returns the
    status word."""
    dev = refs.get_device()
    t = _page_tables(dev, table, lens, refs, page_size)
    return _pages_call(dev, "nls_cache_release", refs, lib().nls_cache_workspace(t, 0), t, _ints(dev, slots), slots.numel())


def cache_reorder(kv, table, lens, refs, parents, fmt: Optional[PageFormat] = None):
    """Every slot s becomes what slot parents[s] (int32 [slots]; -1: nothing) was:
    full pages shared, a parent's last partial page kept by itself or its first
    child and copied for the others, in every layer of kv.  Returns the status
    word."""
    dev = refs.get_device()
    if not (parents.numel() == table.shape[0] and kv.shape[1] == refs.numel()):
        raise AssertionError("parents: one per slot; refs: one per page of kv")
    t = _page_tables(dev, table, lens, refs, _page_size(kv, fmt))
    return _pages_call(dev, "nls_cache_reorder", refs, lib().nls_cache_reorder_workspace(t), _page_pool(dev, kv, fmt), t,
                       _ints(dev, parents))


def cache_compact(kv, table, refs, fmt: Optional[PageFormat] = None):
    """Moves the held pages to the lowest ids, their contents in every layer and
    the table's entries with them.  Returns how many are held, int32 [1]."""
    dev = refs.get_device()
    if kv.shape[1] != refs.numel():
        raise AssertionError("refs: one per page of kv")
    t = _page_tables(dev, table, None, refs, _page_size(kv, fmt))
    return _pages_call(dev, "nls_cache_compact", refs, lib().nls_cache_workspace(t, 0), _page_pool(dev, kv, fmt), t)


def cache_copy_pages(kv, src, dst, fmt: Optional[PageFormat] = None):
    """Page src[i] to page dst[i] (int32) in every layer of kv."""
    dev = kv.get_device()
    if not (dev >= 0 and src.numel() == dst.numel()):
        raise AssertionError("copies: kv on the GPU, src and dst of one length")
    _launch(dev, "nls_cache_copy_pages", _page_pool(dev, kv, fmt), kv.shape[1], _ints(dev, src), _ints(dev, dst), src.numel())


class PagedCache:
    """Keys and values of `slots` contexts in pages: the device counterpart of the
    dense cache of an nimllm context (src/nimllm/model.nim:300-302), for several
    contexts that share one pool.

    kv [layers, pages, 2, kv_heads, page_size, head_dim]; table [slots,
    max_pages], lens [slots] and refs [pages] are int32.  dtype may be a torch
    type, or "q8_0" or "q4_0": blocks of 8 or 4 bits, kv then uint8 [layers,
    pages, page_bytes] in the format `fmt`.  A decoding step is reserve(counts),
    then append and attend layer by layer; nothing of it waits for the device, so
    it can be captured into a graph and replayed."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, slots: int,
                 max_pages: int, dtype=None, device="cuda"):
        import torch

        device = torch.empty(0, device=device).device
        self.fmt = PageFormat(dtype, kv_heads, page_size, head_dim) if isinstance(dtype, str) else None
        if self.fmt is None:
            self.kv = torch.zeros((layers, pages, 2, kv_heads, page_size, head_dim), dtype=dtype or torch.float32,
                                  device=device)
        else:
            self.kv = torch.zeros((layers, pages, self.fmt.page_bytes), dtype=torch.uint8, device=device)
        self.table = torch.full((slots, max_pages), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(slots, dtype=torch.int32, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self.page_size = page_size

    def reserve(self, counts):
        return cache_reserve(self.table, self.lens, self.refs, self.page_size, counts)

    def append(self, layer: int, k, v, starts, q=None, plan=None, slots=None, out=None):
        return cache_append(self.kv[layer], self.table, self.lens, starts, k, v, q=q, plan=plan, slots=slots, out=out,
                            fmt=self.fmt)

    def read(self, layer: int, starts, tokens: int, **kw):
        return cache_read(self.kv[layer], self.table, self.lens, starts, tokens, fmt=self.fmt, **kw)

    def attend(self, layer: int, q, starts, **kw):
        return paged_attention(q, self.kv[layer], self.table, self.lens, starts, fmt=self.fmt, **kw)

    def fork(self, src, dst):
        return cache_fork(self.kv, self.table, self.lens, self.refs, src, dst, fmt=self.fmt)

    def reorder(self, parents):
        return cache_reorder(self.kv, self.table, self.lens, self.refs, parents, fmt=self.fmt)

    def release(self, slots):
        return cache_release(self.table, self.lens, self.refs, slots, self.page_size)

    def compact(self):
        return cache_compact(self.kv, self.table, self.refs, fmt=self.fmt)


# ---------------------------------------------------------------- beam search


def beam_select(logits, scores, ended=None, eog=None, out=None, work=None):
    """The next beams of each group: of all continuations (r, v) of its rows,
    worth scores[r] + ln softmax(logits[r])[v], the best ones in descending order
    (of equal ones the lowest).  logits: float32 [groups * beams, V] (or [groups,
    beams, V]), scores: float32 [groups, beams].  ended (int32 [groups, beams]):
    beams that stand for themselves alone; eog (int32): the ids that end one.

    Returns (parents, tokens, scores, ended), [groups, beams] each: parents are
    rows of `logits`, tokens -1 where a beam had ended or there were too few
    continuations (its score is -infinity then, its parent its own row).  `out`:
    four such tensors; scores and ended may be those given.  `work`: a
    preallocated uint8 workspace of nls_beam_workspace() bytes."""
    import torch

    dev = logits.get_device()
    groups, beams = scores.shape
    vocab = logits.shape[-1]
    if not (dev >= 0 and logits.dtype == torch.float32 and logits.is_contiguous() and
            logits.numel() == groups * beams * vocab):
        raise AssertionError("beams: logits float32 [groups * beams, V] on the GPU, contiguous")
    if not (vocab < 1 << 29 and groups * beams < 1 << 24):
        raise AssertionError("beams: V below 2^29, fewer than 2^24 rows")
    if out is None:
        # (one buffer: an allocation less for each of the others)
        ints = torch.empty((3, groups, beams), dtype=torch.int32, device=logits.device).unbind()
        out = ints[0], ints[1], torch.empty_like(scores), ints[2]
    parents, tokens, worth, over = out
    for x in (scores, worth):
        if not (x.get_device() == dev and x.dtype == torch.float32 and x.is_contiguous() and x.shape == scores.shape):
            raise AssertionError("beams: scores float32 [groups, beams], contiguous, on the logits' device")
    for x in (parents, tokens, over, ended):
        if x is not None and x.shape != scores.shape:
            raise AssertionError("beams: parents, tokens and ended of the scores' shape")
    need = lib().nls_beam_workspace(groups, beams, vocab)
    if work is None or work.numel() < need:
        work = torch.empty(max(need, 1), dtype=torch.uint8, device=logits.device)
    elif not (work.get_device() == dev and work.dtype == torch.uint8 and work.is_contiguous()):
        raise AssertionError("work: uint8, contiguous, on the call's device")
    _launch(dev, "nls_beam_select", logits.data_ptr(), groups, beams, vocab, scores.data_ptr(), _ints(dev, ended),
            _ints(dev, eog), 0 if eog is None else eog.numel(), _ints(dev, parents), _ints(dev, tokens),
            worth.data_ptr(), _ints(dev, over), work.data_ptr(), work.numel())
    return out
