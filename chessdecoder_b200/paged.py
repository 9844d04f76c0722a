"""KV-cache inference with a length of its own per sequence: a pool of pages
(csrc/paged.cu) under the same weights and layer loop as decode.BatchedBackbone.

``BatchedBackbone`` keeps, as the reference does
(chessdecoder/cpp/decoder/batched_backbone.hpp:17-94), one dense cache of one
length for the whole batch and marks which keys count.  Rollouts whose games
have different lengths, end at different times and make room for new ones waste
most of it.  Here a sequence holds just the pages that its tokens fill, and the
rows are bf16, or e4m3 with one power-of-two scale a row (half the bytes that a
step reads).

* ``PagedKVCache``: the pool of every layer, the page tables and lengths (on the
  device, read by the kernels) and the allocator (on the host).
* ``PagedBackbone``: ``prefill`` (prompts into empty sequences), ``step`` (one
  token per active sequence, replayed from a CUDA graph) and ``generate`` (the
  whole loop on the device, with the log-probability, the entropy and the best
  alternatives of every choice).
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import kernels as K
from .decode import HEAD_DIM, _Backbone, _u8


class PagedKVCache:
    """Pages of ``page_size`` rows (a power of two) for ``max_seqs`` sequences of
    up to ``max_len`` tokens.  Tensors (per layer in dimension 0):

    * ``k`` / ``v``: ``dtype`` [L, num_pages, kv_heads, page_size, 64], and for
      float8_e4m3fn ``k_scale`` / ``v_scale`` float8_e8m0fnu
      [L, num_pages, kv_heads, page_size];
    * ``table``: int32 [max_seqs, pages of max_len]; ``lens``: int32 [max_seqs];
      ``start`` / ``count``: where the tokens of the running call begin and how
      many each sequence has.

    ``reserve`` and ``release`` are host calls: they move pages between the free
    list and the sequences and copy the table to the device."""

    def __init__(self, num_layers: int, num_pages: int, max_seqs: int, max_len: int, kv_heads: int,
                 page_size: int = 64, dtype=torch.bfloat16, device="cuda"):
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError("a paged cache is bfloat16 or float8_e4m3fn")
        if page_size < 1 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two")
        if min(num_layers, num_pages, max_seqs, max_len, kv_heads) < 1:
            raise ValueError("num_layers, num_pages, max_seqs, max_len and kv_heads must be positive")
        self.device = torch.device(device)
        self.page_size, self.max_len, self.max_seqs, self.num_pages = page_size, max_len, max_seqs, num_pages
        shape = (num_layers, num_pages, kv_heads, page_size)
        self.k = torch.zeros(*shape, HEAD_DIM, dtype=dtype, device=self.device)
        self.v = torch.zeros_like(self.k)
        self.k_scale = self.v_scale = None
        if dtype == torch.float8_e4m3fn:
            self.k_scale = torch.ones(shape, dtype=torch.uint8, device=self.device).view(torch.float8_e8m0fnu)
            self.v_scale = torch.ones(shape, dtype=torch.uint8, device=self.device).view(torch.float8_e8m0fnu)
        width = -(-max_len // page_size)
        self._table = torch.full((max_seqs, width), -1, dtype=torch.int32)
        self.table = self._table.to(self.device)
        self.lens = torch.zeros(max_seqs, dtype=torch.int32, device=self.device)
        self.start = torch.zeros_like(self.lens)
        self.count = torch.zeros_like(self.lens)
        self._len = [0] * max_seqs
        self._held = [0] * max_seqs  # pages of each sequence: the first entries of its table row
        self._free = list(range(num_pages - 1, -1, -1))

    @property
    def lengths(self):
        """Tokens in each sequence."""
        return list(self._len)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def layer(self, i: int) -> dict:
        """Layer i's pool, as the arguments of K.paged_append / paged_gather / paged_attn."""
        return dict(k_pages=self.k[i], v_pages=self.v[i], table=self.table,
                    k_scale=None if self.k_scale is None else self.k_scale[i],
                    v_scale=None if self.v_scale is None else self.v_scale[i])

    def reserve(self, new: Sequence[int]):
        """Pages for new[b] more tokens of every sequence b.  Raises ValueError,
        and takes nothing, when a sequence would pass max_len or the pool has too
        few pages."""
        if len(new) != self.max_seqs:
            raise ValueError(f"{len(new)} counts for {self.max_seqs} sequences")
        want = []
        for b, n in enumerate(new):
            if n < 0 or self._len[b] + n > self.max_len:
                raise ValueError(f"cache full: sequence {b} has {self._len[b]} + {n} > {self.max_len}")
            want.append(max(-(-(self._len[b] + n) // self.page_size) - self._held[b], 0))
        if sum(want) > len(self._free):
            raise ValueError(f"out of pages: {sum(want)} needed, {len(self._free)} free")
        if not any(want):
            return
        for b, n in enumerate(want):
            for _ in range(n):
                self._table[b, self._held[b]] = self._free.pop()
                self._held[b] += 1
        self.table.copy_(self._table)

    def advance(self, new: Sequence[int]):
        """The host's lengths after a call wrote new[b] tokens (``lens`` itself is
        moved on the device by the call)."""
        for b, n in enumerate(new):
            self._len[b] += n

    def settle(self, lengths: Sequence[int]):
        """Both lengths as they were before a call that raised on its way: it may
        have moved the device's, and the rows that it wrote behind them count no
        more."""
        self._len = list(lengths)
        self.lens.copy_(torch.tensor(self._len, dtype=torch.int32))

    def release(self, seqs):
        """Empties sequences: their pages are free, their length is 0."""
        seqs = [int(b) for b in seqs]
        for b in seqs:
            if not -self.max_seqs <= b < self.max_seqs:
                raise IndexError(f"no sequence {b} of {self.max_seqs}")
        for b in seqs:
            held = self._held[b]
            self._free.extend(reversed(self._table[b, :held].tolist()))
            self._table[b] = -1
            self._held[b] = self._len[b] = 0
        if seqs:
            self.table.copy_(self._table)
            self.lens[torch.tensor(seqs, device=self.device)] = 0


def _check_overrides(ids, ov, om):
    for name, t in (("ov", ov), ("om", om)):
        if t is not None and t.numel() != ids.numel():
            raise ValueError(f"{name} must have a value for each of the {ids.numel()} tokens, has {t.numel()}")


def _flags(active, B):
    if active is None:
        return [1] * B
    flags = [int(bool(a)) for a in (active.reshape(-1).tolist() if torch.is_tensor(active) else active)]
    if len(flags) != B:
        raise ValueError(f"{len(flags)} flags for {B} sequences")
    return flags


class PagedBackbone(_Backbone):
    """The dense ChessDecoder's KV-cache backbone over a PagedKVCache (causal
    attention).  ``batch_size`` sequences of up to ``max_seq_len`` tokens share
    ``num_pages`` pages (default: enough for all of them at full length);
    ``kv_dtype``: torch.bfloat16 or torch.float8_e4m3fn.  A prefill, step or
    generate that raises leaves every sequence with the tokens that it had."""

    def __init__(self, cfg=None, batch_size: int = 1, max_seq_len: Optional[int] = None, num_pages: Optional[int] = None,
                 page_size: int = 64, kv_dtype=torch.bfloat16, **kw):
        self._pool = (num_pages, page_size, kv_dtype)
        super().__init__(cfg, batch_size, max_seq_len, **kw)

    def _make_caches(self):
        num_pages, page_size, dtype = self._pool
        if num_pages is None:
            num_pages = self.B * -(-self.max_len // page_size)
        H = self.cfg.num_heads
        self.cache = PagedKVCache(self.cfg.num_layers, num_pages, self.B, self.max_len, H, page_size, dtype, self.device)
        self._ws = None  # attention workspace, one for every step: they run one after the other
        self._step = None
        self._ends = None  # the last token's row of each sequence, after prompts of different lengths

    @property
    def lengths(self):
        return self.cache.lengths

    def release(self, seqs):
        """Empties sequences, so that prefill can begin others in their place."""
        self.cache.release(seqs)

    def _last_rows(self):
        """... and after prompts the row of each one's last token, not of the padding
        behind it.  (A sequence that took no token in the call has none.)"""
        if self._ends is None:
            return super()._last_rows()
        return self.last_hidden16[torch.arange(self.B, device=self.device), self._ends]

    # -- prompts -------------------------------------------------------------
    def prefill(self, ids, num_real=None, ov=None, om=None):
        """Prompts ids [B, S] into empty sequences, num_real[b] tokens each (host
        integers or a tensor; default S; 0 leaves a sequence as it is, whatever it
        holds).  Returns the final hidden states [B, S, E] (fp32); rows of padding
        are of no use.  The attention reads the rows as the cache holds them, so an
        8-bit cache answers a prompt and its continuation alike."""
        B, S = ids.shape
        c = self.cache
        if B != self.B:
            raise ValueError(f"batch {B} != {self.B}")
        real = [S] * B if num_real is None else [int(n) for n in (
            num_real.tolist() if torch.is_tensor(num_real) else num_real)]
        if len(real) != B or any(n < 0 or n > S for n in real):
            raise ValueError(f"num_real must be {B} counts of 0 .. {S}")
        _check_overrides(ids, ov, om)
        for b, n in enumerate(real):
            if n and c._len[b]:
                raise ValueError(f"prefill needs an empty sequence; {b} holds {c._len[b]} tokens")
        if S == 0:
            return torch.empty(B, 0, self.cfg.embed_dim, device=self.device)
        c.reserve(real)
        before = c.lengths
        try:
            h = self._prompts(ids, real, ov, om)
            self._ends = None if min(real) == S else torch.tensor([max(n - 1, 0) for n in real], device=self.device)
            c.advance(real)
        except BaseException:
            c.settle(before)
            raise
        return h

    def _prompts(self, ids, real, ov, om):
        B, S = ids.shape
        c, dev, E, H = self.cache, self.device, self.cfg.embed_dim, self.cfg.num_heads
        T = B * S
        count = torch.tensor(real, dtype=torch.int32, device=dev)
        c.start.copy_(c.lens)
        c.lens.add_(count)
        pos = self._arange32(S).repeat(B)
        x = self._embed_rows(ids, ov, om)
        # rotated q, and k / v as cached, in the training attention's layout; rows of padding stay 0
        qkv16 = torch.zeros(T, 3 * E, dtype=torch.bfloat16, device=dev)
        k_rows, v_rows = (qkv16[:, i * E:(i + 1) * E].view(B, S, H, HEAD_DIM).transpose(1, 2) for i in (1, 2))
        lse = torch.empty(B * H * S, device=dev)
        # other sequences (count 0) hold other tokens: only the prompts are read back
        seen = torch.where(count > 0, c.lens, 0)

        def attend(i, qkv, ao):
            pool = c.layer(i)
            K.paged_append(qkv, B, S, H, start=c.start, num_new=count, pos=pos, rope=self.rope, q_out=qkv16[:, :E],
                           **pool)
            K.paged_gather(lens=seen, k_out=k_rows, v_out=v_rows, **pool)
            K.attn_fwd(qkv16, ao, lse, B, B, S, H)

        return self._layers_forward(x, B, S, attend)

    def _embed_rows(self, ids, ov, om):
        dev, T = self.device, ids.numel()
        ids = ids.to(device=dev, dtype=torch.int64).reshape(-1).contiguous()
        ov = (torch.zeros(T, device=dev) if ov is None else
              ov.to(device=dev, dtype=torch.float32).reshape(-1).contiguous())
        om = torch.zeros(T, dtype=torch.uint8, device=dev) if om is None else _u8(om, dev).reshape(-1)
        return self._embed(ids, ov, om)

    # -- one token -----------------------------------------------------------
    def _step_body(self, ids, ov, om):
        """One token for every sequence with count 1: lengths, all layers, final
        norm.  Everything it reads or moves is on the device, so it can be replayed."""
        c, B, H = self.cache, self.B, self.cfg.num_heads
        c.start.copy_(c.lens)
        c.lens.add_(c.count)
        x = self._embed_rows(ids, ov, om)
        # sequences that take no token keep whatever is in their row of q: nobody reads their output
        q16 = torch.zeros(B, self.cfg.embed_dim, dtype=torch.bfloat16, device=self.device)

        def attend(i, qkv, ao):
            pool = c.layer(i)
            K.paged_append(qkv, B, 1, H, start=c.start, num_new=c.count, pos=c.start, rope=self.rope, q_out=q16, **pool)
            K.paged_attn(q16, lens=c.lens, out=ao, scale=HEAD_DIM ** -0.5, workspace=self._ws, **pool)

        return self._layers_forward(x, B, 1, attend)

    def _begin(self, flags, n):
        """Room for n tokens of the active sequences; the device's flags."""
        if self._ws is None:
            H = self.cfg.num_heads
            self._ws = torch.empty(K.paged_attn_workspace(self.B, H, H), dtype=torch.uint8, device=self.device)
        self.cache.reserve([n * f for f in flags])
        self.cache.count.copy_(torch.tensor(flags, dtype=torch.int32))

    def step(self, ids, ov=None, om=None, active=None):
        """One token ids [B, 1] for every active sequence, at the position that
        its length says.  Returns the final hidden states [B, 1, E] (fp32; of use for
        active sequences).  Replayed from a CUDA graph after the first call: the
        result is then a static buffer, valid until the next step."""
        if tuple(ids.shape) != (self.B, 1):
            raise ValueError(f"a step takes ids [{self.B}, 1]")
        _check_overrides(ids, ov, om)
        flags = _flags(active, self.B)
        self._begin(flags, 1)
        before = self.cache.lengths
        try:
            if self._step is None or not self.use_graphs:
                h = self._step_body(ids, ov, om)  # eager: every lazy set-up happens outside capture
                if self.use_graphs:
                    self._step = "warm"
            else:
                if self._step == "warm":
                    self._step = _Captured(self)
                h = self._step.replay(self, ids, ov, om)
            self._ends = None
            self.cache.advance(flags)
        except BaseException:
            self.cache.settle(before)
            raise
        return h

    # -- generation ------------------------------------------------------------
    def generate(self, ids, n_steps: int, head: str = "board_head", lut=None, active=None, temperature: float = 0.0,
                 seed: int = 0, top_k: int = 0) -> dict:
        """n_steps tokens of every active sequence from the first input token ids
        [B, 1]: each step takes the ``head`` logits of its hidden state, picks a
        token (argmax at temperature <= 0, otherwise a sample, as
        BatchedBackbone.generate), maps it by ``lut`` (sub-vocabulary index -> token
        id; None: identity) and feeds it back.  The loop is replayed from a CUDA
        graph, without the host.  Returns device tensors: ``ids`` int64 [n, B],
        ``log_probs``, ``entropy`` [n, B] (of the unscaled softmax) and, for
        top_k > 0, ``top_ids`` int64, ``top_log_probs`` [n, B, top_k]: the best
        tokens of each step, the chosen one among them or not."""
        B = self.B
        flags = _flags(active, B)
        n_steps = max(int(n_steps), 0)
        temperature = float(max(temperature, 0.0))
        key = (head, None if lut is None else tuple(int(x) for x in lut), temperature, int(top_k))
        st = self._gen.get(key)
        if st is None:
            st = self._gen[key] = _GenLoop(self, head, lut, temperature, int(top_k))
        out = st.outputs(n_steps)
        if n_steps == 0:
            return out
        st.ids.copy_(ids.reshape(B, 1))
        self._begin(flags, n_steps)
        st.seed.fill_(int(seed) & 0x7FFFFFFFFFFFFFFF)
        st.counter.zero_()
        before = self.cache.lengths
        try:
            for i in range(n_steps):
                if i == 0 or not self.use_graphs:
                    st.body(self)  # eager: every lazy set-up happens outside capture
                else:
                    st.replay(self)
                for name, rows in out.items():
                    rows[i].copy_(getattr(st, name).view_as(rows[i]))
                self._ends = None
                self.cache.advance(flags)
        except BaseException:
            self.cache.settle(before)
            raise
        return out


class _Captured:
    """PagedBackbone.step as a CUDA graph with static inputs.  (It does not hold
    the backbone: a cycle would leave the graph's end to the garbage collector,
    which may run while another graph is being captured, and that ends a capture.)"""

    def __init__(self, bb: PagedBackbone):
        dev, B = bb.device, bb.B
        self.ids = torch.zeros(B, 1, dtype=torch.int64, device=dev)
        self.ov = torch.zeros(B, 1, device=dev)
        self.om = torch.zeros(B, 1, dtype=torch.bool, device=dev)
        self.graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize(dev)
        n0 = K.LAUNCHES[0]
        with torch.cuda.graph(self.graph):
            self.out = bb._step_body(self.ids, self.ov, self.om)
        self.n_launch = K.LAUNCHES[0] - n0  # kernels of the library in one replay
        K.LAUNCHES[0] = n0
        self.out16 = bb.last_hidden16

    def replay(self, bb: PagedBackbone, ids, ov, om):
        self.ids.copy_(ids, non_blocking=True)
        for buf, t in ((self.ov, ov), (self.om, om)):
            if t is None:
                buf.zero_()
            else:
                buf.copy_(t.reshape(buf.shape), non_blocking=True)
        self.graph.replay()
        K.LAUNCHES[0] += self.n_launch
        bb.last_hidden16 = self.out16
        return self.out


class _GenLoop:
    """Static buffers and the captured step of a generation loop."""

    def __init__(self, bb: PagedBackbone, head: str, lut, temperature: float, top_k: int):
        dev, B = bb.device, bb.B
        self.temperature, self.top_k = temperature, top_k
        self.weight, self.bias = bb.store.bf16(f"{head}.weight"), bb.store.param(f"{head}.bias")
        V = self.weight.shape[0]
        if not 0 <= top_k <= min(V, K.MAX_TOP):
            raise ValueError(f"top_k must be 0 .. {min(V, K.MAX_TOP)}")
        self.lut = None if lut is None else torch.as_tensor(list(lut), dtype=torch.int64, device=dev)
        if self.lut is not None and self.lut.numel() != V:
            raise ValueError(f"lut has {self.lut.numel()} entries, head {head} has {V} outputs")
        self.ids = torch.zeros(B, 1, dtype=torch.int64, device=dev)  # the step's input, then its choice
        self.idx = torch.zeros(B, dtype=torch.int64, device=dev)
        self.idx32 = torch.zeros(B, dtype=torch.int32, device=dev)
        self.logits = torch.empty(B, V, device=dev)
        self.log_probs, self.entropy = torch.zeros(B, device=dev), torch.zeros(B, device=dev)
        self.top_idx = torch.zeros(B, top_k, dtype=torch.int32, device=dev)
        self.top_ids = torch.zeros(B, top_k, dtype=torch.int64, device=dev)
        self.top_log_probs = torch.zeros(B, top_k, device=dev)
        self.seed = torch.zeros(1, dtype=torch.int64, device=dev)
        self.counter = torch.zeros(1, dtype=torch.int32, device=dev)
        self.graph = None
        self.n_launch = 0

    def outputs(self, n: int) -> dict:
        names = ["ids", "log_probs", "entropy"] + (["top_ids", "top_log_probs"] if self.top_k else [])
        shape = {name: getattr(self, name) for name in names}
        return {name: torch.empty(n, *(t.shape if name != "ids" else t.shape[:1]), dtype=t.dtype, device=t.device)
                for name, t in shape.items()}

    def body(self, bb: PagedBackbone):
        bb._step_body(self.ids, None, None)
        K.gemm(bb.last_hidden16.reshape(bb.B, -1), self.weight, kind=K.EPI_STORE_F32, out=self.logits, bias=self.bias)
        K.head_select(self.logits, self.idx, temperature=self.temperature, seed=self.seed, counter=self.counter)
        self.idx32.copy_(self.idx)
        K.token_logprobs(self.logits, self.idx32, self.log_probs, entropy=self.entropy,
                         top_ids=self.top_idx if self.top_k else None,
                         top_lp=self.top_log_probs if self.top_k else None)
        if self.lut is None:
            self.ids.copy_(self.idx.view(-1, 1))
            self.top_ids.copy_(self.top_idx)
        else:
            self.ids.copy_(self.lut[self.idx].view(-1, 1))
            if self.top_k:
                self.top_ids.copy_(self.lut[self.top_idx.long()])

    def replay(self, bb: PagedBackbone):
        if self.graph is None:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize(bb.device)
            n0 = K.LAUNCHES[0]
            with torch.cuda.graph(graph):
                self.body(bb)
            self.n_launch = K.LAUNCHES[0] - n0
            K.LAUNCHES[0] = n0
            self.graph, self.out16 = graph, bb.last_hidden16
        self.graph.replay()
        K.LAUNCHES[0] += self.n_launch
        bb.last_hidden16 = self.out16
