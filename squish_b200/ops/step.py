"""Serving-step operators: the step's layout on the device, low-rank adapters of many requests,
scored expert routing and sampling from given uniform numbers.

Like the wrappers in :mod:`.kernels`, every call launches on the current CUDA stream and can be
captured in a CUDA graph; with the output provided none allocates, but :func:`lora_add` with more
than 512 rows (a scratch of 4 bytes per row and rank) and :func:`lora_linear` with ``silu_mul`` (the
projection before the activation), from torch's caching allocator. No scratch memory is shared
between calls, so calls on several streams, and captured graphs, do not disturb one another.
"""
from __future__ import annotations

import torch

from .._ext import native
from .kernels import Int4Weight, Workspace, _count, w4a16_linear, workspace

def _status(ws: Workspace | None, t: torch.Tensor, name: str) -> torch.Tensor:
    """Status word of the given workspace, or of the one of the tensor's device."""
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    return (ws or workspace(t.device)).status


LAYOUT_TILE = 32  # queries per attention tile (models.decoder.prefill_tiles)


class StepLayout:
    """Device buffers of one step's layout, for up to ``max_seqs`` sequences, ``max_tokens`` tokens
    and ``max_tiles`` attention tiles (default: enough for any step of that size).

    After :func:`step_layout` over B sequences with T tokens and N tiles (all int32):

    * ``q_start`` [B + 1]: first row of every sequence, then T; ``kv_len`` [B]: cache length after
      the step; ``last_row`` [B]: row of the sequence's last token, -1 for a resting sequence
    * ``positions``, ``slots``, ``token_seq`` [max_tokens]: position, cache slot and sequence of
      every token; rows from T on are padding (position 0, slot -1: not stored, sequence -1)
    * ``tile_seq``, ``tile_q0`` [max_tiles]: the attention tiles; entries from N on are padding
      (sequence 0, a query past its end: the attention kernels skip them), so a captured launch over
      max_tiles covers every step
    * ``totals`` [3]: T, pages taken from the free list, N
    """

    def __init__(self, max_seqs: int, max_tokens: int, max_tiles: int | None = None, device="cuda",
                 tile: int = LAYOUT_TILE):
        if max_seqs < 1 or max_tokens < 1:
            raise ValueError("a step layout holds at least one sequence and one token")
        if tile < 1:
            raise ValueError("an attention tile has at least one query")
        if max_tiles is None:
            max_tiles = max_tokens // tile + min(max_seqs, max_tokens)
        self.max_seqs, self.max_tokens, self.max_tiles, self.tile = max_seqs, max_tokens, max_tiles, tile
        # one buffer (one argument of the launch), each row padded to a multiple of four
        sizes = (max_seqs + 1, max_seqs, max_seqs, 3, max_tokens, max_tokens, max_tokens, max_tiles, max_tiles)
        self.buf = torch.zeros(sum((n + 3) // 4 * 4 for n in sizes), dtype=torch.int32, device=device)
        rows, at = [], 0
        for n in sizes:
            rows.append(self.buf[at:at + n])
            at += (n + 3) // 4 * 4
        (self._q_start, self._kv_len, self._last_row, self.totals, self.positions, self.slots, self.token_seq,
         self.tile_seq, self.tile_q0) = rows
        self._narrow(max_seqs)

    def _narrow(self, b: int) -> None:
        if b > self.max_seqs:
            raise ValueError(f"a step of {b} sequences in a layout of {self.max_seqs}")
        self.seqs = b
        self.q_start, self.kv_len, self.last_row = self._q_start[:b + 1], self._kv_len[:b], self._last_row[:b]


def step_layout(ctx_len: torch.Tensor, q_len: torch.Tensor, block_tables: torch.Tensor, free_pages: torch.Tensor,
                page_size: int, out: StepLayout, ws: Workspace | None = None) -> StepLayout:
    """Positions, cache slots, sequence bounds and attention tiles of a step, from ``ctx_len`` [B]
    (tokens already cached) and ``q_len`` [B] (tokens of this step, 0 = resting), on the device.

    Row b of ``block_tables`` [B, W] holds the sequence's ceil(ctx / page_size) pages; the pages its
    new tokens need are taken from the front of ``free_pages``, in sequence order, and appended to
    the row (``out.totals[1]`` of them in all). A token whose page is -1 (given back) gets slot -1.

    What does not fit is not written and records SQ_ERR_BOUNDS in the workspace status: tokens past
    the buffers, pages past the row's width or the end of the free list (their tokens get slot -1),
    tiles past ``max_tiles`` (their queries are not computed).
    A sequence whose tokens do not all fit rests: its ``kv_len`` is ``ctx_len`` (at most what its row
    of the table can hold), its ``last_row`` -1, and its tiles are padding, so that attention reads no
    page that is not the sequence's. A sequence with a length below 0 or of 2^30 tokens and more
    counts as resting and records it as well. The lengths
    may not be rows of ``out`` itself (copy ``out.kv_len`` to make it the next step's ``ctx_len``), nor
    they or the free list part of the tables."""
    b = ctx_len.numel()
    if b != out.seqs:
        out._narrow(b)
    native().step_layout(ctx_len, q_len, block_tables, free_pages, page_size, out.tile, out.buf, out.max_seqs,
                         out.max_tokens, out.max_tiles, _status(ws, ctx_len, "ctx_len"))
    _count()
    return out


# ----------------------------------------------------------------------------- sampling
def sample_uniform(logits: torch.Tensor, uniforms: torch.Tensor, out_tokens: torch.Tensor,
                   temperature: torch.Tensor | None = None, top_p: torch.Tensor | None = None,
                   top_k: torch.Tensor | None = None, min_p: torch.Tensor | None = None,
                   allow_mask: torch.Tensor | None = None, out_logprob: torch.Tensor | None = None) -> torch.Tensor:
    """One token per row of bf16 ``logits`` [B, V], a function of the row and of its number in
    ``uniforms`` (float32 [B], in [0, 1)): inverse-transform sampling over the tokens in descending
    order of logit, the lower index first among equals. Filters as in :func:`sample` (per row:
    min-p, then top-k, then top-p over the full softmax), with exactly ``top_k`` tokens and exactly
    the shortest top-p prefix when logits tie; at least one token stays. temperature <= 0 (or none):
    the first largest logit. ``allow_mask`` int32 [B, ceil(V / 32)]: bit set = allowed. A row without
    an allowed finite logit gives token -1 and log-probability -inf. ``out_logprob``: log-probability
    of the token among the kept ones (0 for greedy rows). The repetition penalty of :func:`sample`
    is not part of it: apply it to the logits."""
    native().sample_uniform(logits, uniforms, out_tokens, temperature, top_p, top_k, min_p, allow_mask, out_logprob)
    _count()
    return out_tokens


# ----------------------------------------------------------------------------- scored routing
def moe_route_scored(logits: torch.Tensor, top_k: int, ids: torch.Tensor, weights: torch.Tensor,
                     score: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
                     top_groups: int | None = None, group_score: str = "max", renorm: bool = True,
                     scale: float = 1.0) -> None:
    """Router of a MoE layer: ``ids`` (int32 [T * top_k], in order of choice) and ``weights`` (float32)
    from ``logits`` [T, E] (bf16 or float32, E <= 512).

    s = softmax or sigmoid of the logits; the choice is made on s + ``bias`` (float32 [E], a load
    balance correction that does not enter the weights), among the experts of the ``top_groups``
    best of ``groups`` equal groups (ranked by their best value, ``group_score="max"``, or by the
    sum of their two best, ``"top2"``); equal values go to the lower index. weights = s at the chosen
    experts, divided by their sum when ``renorm``, times ``scale``. A NaN logit counts as -inf; a row
    whose chosen scores are all zero gets weights 0."""
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f"score must be 'softmax' or 'sigmoid', not {score!r}")
    if group_score not in ("max", "top2"):
        raise ValueError(f"group_score must be 'max' or 'top2', not {group_score!r}")
    native().moe_route_scored(logits, top_k, ids, weights, score == "sigmoid", bias, groups,
                              groups if top_groups is None else top_groups, group_score == "top2", renorm, scale)
    _count()


# ----------------------------------------------------------------------------- adapters
def fuse_lora(parts: list[tuple[torch.Tensor, torch.Tensor] | None], sizes: list[int], k: int | None = None,
              interleave: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """One (A [r, K], B [N, r]) pair for a fused projection whose output rows are the parts' rows
    one after another (``sizes`` of them): the ranks add up (to 128 at most for a :class:`LoraPool`: q, k
    and v of rank 42) and B is block-diagonal. ``interleave``:
    two parts of equal size, gate and up, in [gate 64 | up 64] row blocks (the layout of the fused
    gate_up weight, sizes padded to a multiple of 64). A part may be None (no adapter there)."""
    if len(parts) != len(sizes):
        raise ValueError("one size per part")
    live = [p for p in parts if p is not None]
    if not live and k is None:
        raise ValueError("no adapted part: give k")
    for p, n in zip(parts, sizes):
        if p is not None and (p[0].shape[0] != p[1].shape[1] or p[1].shape[0] != n):
            raise ValueError(f"an adapter part needs A [r, K] and B [{n}, r]")
    ref = live[0][0] if live else torch.zeros(0, k)
    a = torch.cat([p[0] for p in live]) if live else ref
    r = a.shape[0]
    rows, c = [], 0
    for p, n in zip(parts, sizes):
        b = torch.zeros(n, r, dtype=ref.dtype, device=ref.device)
        if p is not None:
            b[:, c:c + p[1].shape[1]] = p[1]
            c += p[1].shape[1]
        rows.append(b)
    if not interleave:
        return a, torch.cat(rows)
    if len(rows) != 2 or sizes[0] != sizes[1]:
        raise ValueError("gate and up have equal sizes")
    f = (sizes[0] + 63) // 64 * 64
    g, u = (torch.cat([b, b.new_zeros(f - b.shape[0], r)]).view(f // 64, 64, r) for b in rows)
    return a, torch.stack([g, u], 1).reshape(2 * f, r)


class LoraPool:
    """Adapters of one projection [N, K], resident on the device: ``slots`` of them, each A [r, K],
    B [N, r] (r <= ``max_rank`` <= 128) and a scale, in bf16, zero-padded to the pool's rank. The
    same slot numbers name a request's adapter in every projection's pool.

    :func:`lora_add` picks its launch for the most tiles that the rows may make, one per slot, so a
    pool much larger than what a step uses costs time (B200, 5 adapters in a pool of 16 / 256 / 1024 slots,
    us: 512 rows, 3584 x 4608, rank 16 8.6 / 12 / 19, 3584 x 37888 with SiLU*up 32 / 85 / 164; 2048 rows 18 /
    27 / 28 and 58 / 68 / 68; 64 rows over 16 adapters, 3584 x 4608 6.5 in each)."""

    def __init__(self, slots: int, k: int, n: int, max_rank: int, device="cuda"):
        if slots < 1 or slots > 1024:
            raise ValueError("an adapter pool has 1..1024 slots")
        if max_rank < 1 or max_rank > 128:
            raise ValueError("adapter rank must be in 1..128")
        if k < 8 or n < 8 or k % 8 or n % 8:
            raise ValueError("k and n must be positive multiples of 8")
        r = next(v for v in (16, 32, 64, 128) if v >= max_rank)
        self.slots, self.k, self.n, self.max_rank = slots, k, n, max_rank
        self.a = torch.zeros(slots, r, k, dtype=torch.bfloat16, device=device)
        self.b = torch.zeros(slots, n, r, dtype=torch.bfloat16, device=device)
        self.rank = torch.zeros(slots, dtype=torch.int32, device=device)
        self.scale = torch.zeros(slots, dtype=torch.float32, device=device)
        self._filled = [0] * slots  # ranks of a slot that may hold something

    def load(self, slot: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """Put an adapter (A [r, K], B [N, r]; ``scale``: usually alpha / r) into a slot, in the
        current stream's order."""
        r = a.shape[0]
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} outside 0..{self.slots - 1}")
        if a.dim() != 2 or b.dim() != 2 or a.shape[1] != self.k or tuple(b.shape) != (self.n, r):
            raise ValueError(f"an adapter here is A [r, {self.k}] and B [{self.n}, r], not "
                             f"{tuple(a.shape)} and {tuple(b.shape)}")
        if not 1 <= r <= self.max_rank:
            raise ValueError(f"rank {r} outside 1..{self.max_rank}")
        if self._filled[slot] > r:  # a smaller rank leaves nothing of the one before it
            self.a[slot, r:].zero_()
            self.b[slot, :, r:].zero_()
        self._filled[slot] = r
        self.a[slot, :r].copy_(a)
        self.b[slot, :, :r].copy_(b)
        self.rank[slot].fill_(r)
        self.scale[slot].fill_(scale)

    def clear(self, slot: int) -> None:
        """Empty a slot: rows that name it get no adapter."""
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} outside 0..{self.slots - 1}")
        self.rank[slot].fill_(0)


class LoraPlan:
    """A step's rows sorted by adapter slot and cut into tiles (:func:`lora_plan`), shared by every
    projection of the step."""

    def __init__(self, rows: int, slots: int, device):
        # tiles of 16 rows while adapters have few rows each, of 128 for prefill: a tile reads its
        # adapter once, so wider tiles re-read less (from L2) but leave more of themselves empty.
        # (The rule does not know how many adapters the rows name: one request's chunk of up to 512 rows takes
        # the 16-row tiles too, and is slower for it.) Measured on a B200 with 16 / 128, us: 3584 x 3584 rank 16, 16 adapters: 512 rows 9.8 / 12.5,
        # 1024 rows 12.4 / 13.4; 4096 x 6144 rank 64, 16 adapters: 512 rows 19.4 / 23.3, 1024 rows
        # 24.7 / 23.8, one adapter: 256 rows 14.4 / 11.1, 512 rows 20.0 / 12.5, 1024 rows 36.6 / 17.1
        self.tile_rows = 16 if rows <= 512 else 128
        self.rows, self.slots = rows, slots
        self.max_tiles = -(-rows // self.tile_rows) + min(slots + 1, rows)
        i32 = dict(dtype=torch.int32, device=device)
        self.order = torch.empty(rows, **i32)
        self.tiles = torch.empty(self.max_tiles, 4, **i32)
        self.num_tiles = torch.zeros(1, **i32)


def lora_plan(row_slots: torch.Tensor, slots: int, out: LoraPlan | None = None,
              ws: Workspace | None = None) -> LoraPlan:
    """Plan of a step from the adapter slot of every row (int32 [M], -1 = no adapter), by one CTA (B200, 16 /
    1024 slots, us: 64 rows 2.5 / 8.8, 2048 rows 3.9 / 11, 8185 rows 8.0 / 18). ``out``: a plan
    of the same size to refill (CUDA graphs). A slot outside [-1, slots) counts as none and records
    SQ_ERR_BOUNDS in the workspace status."""
    m = row_slots.numel()
    if out is None:
        out = LoraPlan(m, slots, row_slots.device)
    elif out.rows != m or out.slots != slots:
        raise ValueError(f"a plan for {out.rows} rows and {out.slots} slots, not {m} and {slots}")
    native().lora_plan(row_slots, slots, out.tile_rows, out.order, out.tiles, out.num_tiles,
                       _status(ws, row_slots, "row_slots"))
    _count()
    return out


def lora_add(x: torch.Tensor, pool: LoraPool, plan: LoraPlan, y: torch.Tensor, out: torch.Tensor | None = None,
             silu_mul: bool = False, ws: Workspace | None = None) -> torch.Tensor:
    """out[t] = y[t] + scale_s B_s (A_s x[t]) for row t with adapter slot s, out[t] = y[t] without
    one; x [M, K], y [M, N] bf16. ``out`` may be y itself. With ``silu_mul`` the columns of y are
    interleaved gate/up blocks of 64 and out = silu(gate) * up has N/2 columns. Sums are fp32, ``out``
    is rounded once. Where A_s x[t] is not finite the row may hold NaN for an infinity; other rows do
    not notice."""
    if out is None:
        out = torch.empty((x.shape[0], pool.n // 2 if silu_mul else pool.n), dtype=torch.bfloat16, device=x.device)
    native().lora_add(x, pool.a, pool.b, pool.rank, pool.scale, y, out, plan.order, plan.tiles, plan.num_tiles,
                      plan.tile_rows, plan.slots, plan.max_tiles, silu_mul, _status(ws, x, "x"))
    _count()
    return out


def lora_linear(x: torch.Tensor, w: Int4Weight, pool: LoraPool, plan: LoraPlan, out: torch.Tensor | None = None,
                residual: torch.Tensor | None = None, silu_mul: bool = False,
                ws: Workspace | None = None) -> torch.Tensor:
    """:func:`w4a16_linear` with the rows' adapters added (before the SiLU*up epilogue). The projection
    (with the residual) is rounded to bf16 before the adapters are added, and their sum again. With
    ``silu_mul`` that holds for rows without an adapter as well: :func:`w4a16_linear` alone keeps gate and
    up in fp32, so such a row may differ from it by those roundings."""
    if not silu_mul:
        y = w4a16_linear(x, w, out=out, residual=residual, ws=ws)
        return lora_add(x, pool, plan, y, out=y, ws=ws)
    if residual is not None:
        raise ValueError("a residual cannot follow the SiLU*up epilogue")
    y = w4a16_linear(x, w, ws=ws)
    return lora_add(x, pool, plan, y, out=out, silu_mul=True, ws=ws)
