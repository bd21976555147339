"""The Qwen3-TTS talker decode-attention call site of the sokutou engine, on the B200 kernel.

Mirrors the attention state of `Qwen3Kernels` (qwen3/kernels.py:483-706): the per-layer KV caches
(HF StaticCache tensors `[nkv][max_cache][128]`, qwen3/kernels.py:702-705), the RoPE table
(qwen3/kernels.py:473-477), the device-side position (qwen3/fast.py:102) and the per-layer launch
of qwen3/kernels.py:622-624, plus the caller-owned split-KV workspace the B200 kernel needs.
"""

from __future__ import annotations

import torch

from . import ops


def rope_table(max_len: int, theta: float, hd: int = 128, device=None) -> torch.Tensor:
    """float32 (max_len, hd) = [cos(pos·f) | sin(pos·f)] with f = theta^(-2i/hd) computed in float32
    as transformers' default rope init does (qwen3/kernels.py:473-477)."""
    inv = 1.0 / (theta ** (torch.arange(0, hd, 2, dtype=torch.int64, device=device).float() / hd))
    f = torch.arange(max_len, device=device, dtype=torch.float32)[:, None] * inv[None, :]
    return torch.cat([f.cos(), f.sin()], dim=1).contiguous()


class TalkerAttention:
    """KV caches, RoPE table, position and workspace of one talker stack.

    `attn(layer, qkv, qn, kn, out, pos_add=0)` runs one layer's decode attention exactly where
    `_layers` launches the reference kernel; the position is read on the device from `self.pos`
    (advance it with `self.pos.add_(1)` inside the captured frame, qwen3/kernels.py:692).
    """

    def __init__(self, n_layers: int, nq: int, nkv: int, max_len: int, theta: float, eps: float, device,
                 cache_dtype: torch.dtype = torch.bfloat16, hd: int = 128, use_pos: bool = True):
        self.n_layers, self.nq, self.nkv, self.hd, self.max_len, self.eps = n_layers, nq, nkv, hd, max_len, eps
        self.k = torch.zeros((n_layers, nkv, max_len, hd), dtype=cache_dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.rope = rope_table(max_len, theta, hd, device)
        self.pos = torch.zeros((1,), dtype=torch.int64, device=device) if use_pos else None
        self.ws = ops.decode_workspace(max_len, nq, nkv, device, hd, cache_dtype)
        self.block_ws = ops.decode_block_workspace(max_len, nq, nkv, device, hd)

    def attn(self, layer: int, qkv: torch.Tensor, qn: torch.Tensor, kn: torch.Tensor, out: torch.Tensor,
             pos_add: int = 0, kv_stable: bool = False) -> torch.Tensor:
        """kv_stable: the kernel launched just before writes neither self.pos nor this layer's cache (true
        after the layer's qkv projection; false right after the position advance)."""
        return ops.decode_attention(qkv, qn, kn, self.eps, self.rope, self.k[layer], self.v[layer], self.pos, pos_add,
                                    self.max_len, self.nq, self.nkv, out, self.ws, kv_stable)

    def block(self, layer: int, h: torch.Tensor, in_norm: torch.Tensor, eps_in: float, w_qkv: torch.Tensor,
              qn: torch.Tensor, kn: torch.Tensor, w_o: torch.Tensor, pos_add: int = 0,
              kv_stable: bool = False) -> torch.Tensor:
        """The layer's whole attention block — rms_gemv(qkv), the decode attention and gemv(o) into the
        residual h (qwen3/kernels.py:619-624) — in one launch; h (fp32 [hidden]) is updated in place."""
        return ops.decode_attention_block(h, in_norm, eps_in, w_qkv, qn, kn, self.eps, self.rope, self.k[layer],
                                          self.v[layer], self.pos, pos_add, self.max_len, self.nq, self.nkv, w_o,
                                          self.block_ws, kv_stable)


class TalkerGroup:
    """R decode slots of one talker stack behind one shared prefix (a voice prompt decoded once), with
    optionally bounded caches. Not in the reference, which serves one request at a time (README.md:186).

    prefix: (k, v), each (n_layers, nkv, P, hd) in the cache dtype — views of another stack's caches will do,
    e.g. (ta.k[:, :, :P], ta.v[:, :, :P]) of a TalkerAttention that has taken the prompt. `k`, `v`
    (n_layers, R, nkv, max_len, hd) hold each slot's own rows; `pos` and `rows` (int64, R) its position (-1:
    idle) and own rows, read on the device, so one captured step serves all steps. track_mass keeps every
    own row's attention weight (`mass`, float32) for `evict`. n_pos: rows of the RoPE table (default P +
    max_len; more where eviction lets a slot outlive its cache).

    `attn(layer, qkv, qn, kn, out)` runs one layer for all slots, `advance()` moves the live ones on by one
    position, `evict(keep, ...)` brings every layer's caches down to `keep` own rows, in place.
    """

    def __init__(self, n_layers: int, R: int, nq: int, nkv: int, max_len: int, theta: float, eps: float, device,
                 prefix: tuple[torch.Tensor, torch.Tensor] | None = None, cache_dtype: torch.dtype = torch.bfloat16,
                 hd: int = 128, n_pos: int | None = None, track_mass: bool = False,
                 act_dtype: torch.dtype = torch.float32):
        self.n_layers, self.R, self.nq, self.nkv, self.hd, self.max_len, self.eps = n_layers, R, nq, nkv, hd, max_len, eps
        self.prefix_len = 0 if prefix is None else prefix[0].shape[2]
        self.k = torch.zeros((n_layers, R, nkv, max_len, hd), dtype=cache_dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.mass = torch.zeros((n_layers, R, nkv, max_len), device=device) if track_mass else None
        self.rope = rope_table(n_pos or self.prefix_len + max_len, theta, hd, device)
        self.pos = torch.full((R,), -1, dtype=torch.int64, device=device)
        self.rows = torch.zeros((R,), dtype=torch.int64, device=device)
        self._live = torch.zeros((R,), dtype=torch.int64, device=device)
        ws = ops.shared_decode_workspace(R, nq, nkv, max_len, self.prefix_len, device, hd, cache_dtype, track_mass)
        kp, vp = prefix if prefix is not None else (None, None)
        self._plans = [ops.shared_decode_plan(self.k[i], self.v[i], self.pos, self.rope, nq, eps, rows=self.rows,
                                              Kp=None if kp is None else kp[i], Vp=None if vp is None else vp[i],
                                              mass=None if self.mass is None else self.mass[i], qkv_dtype=act_dtype,
                                              out_dtype=act_dtype, workspace=ws) for i in range(n_layers)]
        self._evict_plans: dict[tuple[int, int, int], ops.CacheEvictPlan] = {}
        self._evict_ws = None  # of all budgets: a step evicts by one

    def start(self, slot: int, rows: int = 0) -> None:
        """A request takes the slot, `rows` own rows of its caches already filled (by a prefill, or a copy); their
        weights count from zero."""
        if not 0 <= slot < self.R or not 0 <= rows < self.max_len:
            raise ValueError(f"slot {slot} of {self.R}, {rows} rows of {self.max_len}")
        if rows and self.mass is not None:
            self.mass[:, slot, :, :rows] = 0
        self.pos[slot], self.rows[slot], self._live[slot] = self.prefix_len + rows, rows, 1

    def stop(self, slot: int) -> None:
        """The slot's request has ended: the slot is idle until the next start."""
        if not 0 <= slot < self.R:
            raise ValueError(f"slot {slot} of {self.R}")
        self.pos[slot], self.rows[slot], self._live[slot] = -1, 0, 0

    def attn(self, layer: int, qkv: torch.Tensor, qn: torch.Tensor, kn: torch.Tensor,
             out: torch.Tensor | None = None) -> torch.Tensor:
        return ops.decode_attention_shared(self._plans[layer], qkv, qn, kn, out)

    def advance(self) -> None:
        self.pos.add_(self._live)
        self.rows.add_(self._live)

    def evict(self, keep: int, first: int = 0, recent: int = 0) -> None:
        """Every layer's caches of every slot that holds more than `keep` own rows, down to `keep`: the `first`
        first and `recent` last rows and the most attended of the others. Positions go on as they were."""
        if self.mass is None:
            raise ValueError("evict needs track_mass=True")
        key = (keep, first, recent)
        if key not in self._evict_plans:
            args = (self.k, self.v, self.mass, self.rows)
            if self._evict_ws is None:
                self._evict_ws = ops.cache_evict_plan(*args, self.max_len).workspace
            self._evict_plans[key] = ops.cache_evict_plan(*args, keep, first, recent, workspace=self._evict_ws)
        ops.cache_evict(self._evict_plans[key])
