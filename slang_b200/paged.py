"""Serving several sequences over paged key-value caches.

``PagedRunner`` is ``runner.Runner``'s decode and prefill for a batch whose
caches are pages: all prompts of a batch go through the layers together, packed
end to end (``kv_append_paged`` and ``attn_prefill_packed``), each decode step
appends one token per sequence and attends over its pages (``attn_decode_paged``),
and the next tokens are drawn from the logits with per-sequence settings
(``sample``).  The projections are the same fused GEMMs as ``Runner``'s batched
path (f16 activations); K and V are held in f16, half the bytes of ``Runner``'s
f32 caches, and a sequence takes the pages its length needs.

    dm = runner.DeviceModel(model, "cuda:0", max_seq=4096)
    r = PagedRunner(dm, batch=3, n_pages=256, page_size=16)
    tokens = r.generate([p0, p1, p2], steps=64, temperature=0.8, top_p=0.95, seeds=[1, 2, 3])
"""
from __future__ import annotations

import torch

from . import _lib
from . import kernels as kern

_F16, _F32 = _lib.SB_F16, _lib.SB_F32


class PagedRunner:
    """State of up to ``batch`` sequences of ``dm`` over ``n_pages`` pages of ``page_size``
    tokens per layer.  Layers may differ in head_dim (64, 128 or 256), share another
    layer's K/V and attend over a sliding window; per-layer embeddings are not served.

    The batch is fixed from ``prefill`` to the end.  Up to ``GEMV_ROWS`` sequences are
    sampled from f32 logits, more from f16 ones, so a request may draw another token in
    a larger batch.  All work runs on the runner's own stream, behind the caller's."""

    GEMV_ROWS = 8  # up to this many rows the lm_head is the GEMV with f32 logits, above it the GEMM with f16 ones

    def __init__(self, dm, batch: int, n_pages: int, page_size: int = 16):
        if dm.ple is not None:
            raise ValueError("per-layer embeddings run on Runner(fused=False, proj='gemv')")
        specs = [L["spec"] for L in dm.layers]
        if any(sp["hd"] not in (64, 128, 256) for sp in specs):
            raise ValueError("packed prompts take head_dim 64, 128 or 256; Runner serves the others")
        if batch < 1 or n_pages < 1:
            raise ValueError("batch and n_pages must be positive")
        self.dm, self.B, self.page_size, self.n_pages = dm, batch, page_size, n_pages
        cfg = dm.cfg
        self.H, self.nh, self.eps, self.vocab = cfg["hidden"], cfg["n_heads"], float(cfg["eps"]), cfg["vocab"]
        self.softcap = float(cfg.get("softcap") or 0.0)
        dev = dm.device
        # all work runs on a stream of the runner's own, and so do the fills of its buffers; what the
        # caller's stream still has to do (the model's weights) comes before
        self.stream = torch.cuda.Stream(device=dev)
        with self._own_stream():
            self._allocate(specs, batch, n_pages, page_size)
        self.free = list(range(n_pages))
        # tokens of each sequence behind its prefill, decode steps since then and how many more there is room for
        self.lens, self.taken, self.left = [0] * batch, 0, 0
        self.graph = None

    def _own_stream(self):
        """The runner's stream as the current one, behind all that the caller's stream has been given so far."""
        self.stream.wait_stream(torch.cuda.current_stream(self.dm.device))
        return torch.cuda.stream(self.stream)

    def _allocate(self, specs, batch: int, n_pages: int, page_size: int) -> None:
        dm, dev = self.dm, self.dm.device
        self.caches = []
        for sp in specs:  # a KV-shared layer holds its source layer's cache
            self.caches.append(kern.PagedKV.allocate(n_pages, page_size, 1, sp["hd"], torch.float16, dev)
                               if sp["own"] else self.caches[sp["src"]])
        self.max_pages = -(-dm.max_seq // page_size)
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
        self.table = torch.full((batch, self.max_pages), -1, dtype=torch.int32, device=dev)
        self.pos, self.cur, self.tok, self.history = i32(batch), i32(batch), i32(batch), i32(batch, dm.max_seq)
        self.temperature = torch.zeros(batch, device=dev)
        self.top_k, self.top_p, self.min_p = i32(batch), torch.ones(batch, device=dev), torch.zeros(batch, device=dev)
        self.seeds = torch.zeros(batch, dtype=torch.int64, device=dev)
        # one workspace per shape of attention: the calls follow each other on one stream
        self.attn_ws = {sp["hd"]: kern.attn_decode_paged_workspace(c, self.nh, batch) for sp, c in zip(specs, self.caches)}

    # ------------------------------------------------------------------ requests
    def set_sampling(self, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0, seeds=None) -> None:
        """Sampling settings, each a number for all sequences or one per sequence;
        temperature 0 is greedy.  They may change between steps."""
        with self._own_stream():
            new = []
            for buf, v in ((self.temperature, temperature), (self.top_k, top_k), (self.top_p, top_p),
                           (self.min_p, min_p), (self.seeds, 0 if seeds is None else seeds)):
                if isinstance(v, torch.Tensor) and v.is_cuda:
                    v.record_stream(self.stream)  # its memory stays until this stream has read it
                v = torch.as_tensor(v, dtype=buf.dtype)
                if v.dim() > 1 or (v.dim() and v.numel() != self.B):
                    raise ValueError(f"a setting must be one number or {self.B}")
                new.append((buf, v))
            for buf, v in new:
                buf.copy_(v.expand(self.B))

    def _reserve(self, lens, extra: int) -> int:
        """Pages for each sequence's prompt and ``extra`` more tokens; the last batch's go back.  Returns
        the decode steps that there is room for: a step appends the token that the one before drew,
        and its own goes into the history."""
        need = [-(-(n + extra) // self.page_size) for n in lens]
        if sum(need) > self.n_pages:
            raise ValueError(f"{sum(need)} pages needed, the caches have {self.n_pages}")
        self.free = list(range(self.n_pages))
        rows = torch.full((self.B, self.max_pages), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            rows[b, :n] = torch.tensor([self.free.pop() for _ in range(n)], dtype=torch.int32)
        self.table.copy_(rows)
        self.lens, self.taken, self.left = [n + 1 for n in lens], 0, 0
        return min(min(p * self.page_size - n, self.dm.max_seq - n - 1) for p, n in zip(need, lens))

    # ------------------------------------------------------------------ layers
    def _layers(self, x: torch.Tensor, m: int, attend) -> torch.Tensor:
        """All layers over m rows of the residual stream x (f32, in place); ``attend(li, L, qkv)``
        appends a layer's rows and returns the attention output.  Returns (final hidden f32, f16)."""
        dm, H, s = self.dm, self.H, kern._stream()
        f16 = lambda n: torch.empty(m, n, dtype=torch.float16, device=x.device)  # noqa: E731
        h16, out32 = f16(H), torch.empty(m, H, device=x.device)
        _lib.call("sb_add_rmsnorm", x.data_ptr(), None, _F32, None, dm.layers[0]["in_norm"].data_ptr(), x.data_ptr(),
                  None, h16.data_ptr(), m, H, self.eps, s)
        for li, L in enumerate(dm.layers):
            sp, last = L["spec"], li + 1 == len(dm.layers)
            proj = lambda A, key, **kw: kern.gemm_q4(A, *L[key], bits=L["bits"][key],  # noqa: E731
                                                     workspace=self._gemm_ws(m, L[key], A.shape[1]), **kw)
            attn = attend(li, L, proj(h16, "qkv")).reshape(m, sp["qd"])
            o = proj(attn, "o")
            _lib.call("sb_add_rmsnorm", x.data_ptr(), o.data_ptr(), _F16, L["post_attn_norm"].data_ptr(),
                      L["pre_ffn_norm"].data_ptr(), x.data_ptr(), None, h16.data_ptr(), m, H, self.eps, s)
            d = proj(proj(h16, "gu", geglu=True), "down")
            nxt = dm.final_norm if last else dm.layers[li + 1]["in_norm"]
            _lib.call("sb_add_rmsnorm", x.data_ptr(), d.data_ptr(), _F16, L["post_ffn_norm"].data_ptr(), nxt.data_ptr(),
                      x.data_ptr(), out32.data_ptr() if last else None, h16.data_ptr(), m, H, self.eps, s)
        return out32, h16

    def _gemm_ws(self, m: int, w, k: int):
        """Split-K scratch of one projection, from the stream's own allocator pool."""
        n = kern.gemm_q4_workspace_size(m, w[0].shape[0], k)
        return torch.empty(max(n // 4, 4), dtype=torch.float32, device=self.dm.device)

    def _append(self, li: int, L, qkv, pos, seq, k_out=None, v_out=None) -> torch.Tensor:
        """The layer's rotated queries; a layer that owns its K/V also appends them."""
        sp = L["spec"]
        if sp["own"]:
            return kern.kv_append_paged(qkv, self.caches[li], self.table, pos, L["cos"], L["sin"], self.nh, seq=seq,
                                        q_norm=L["q_norm"], k_norm=L["k_norm"], v_norm=True, eps=self.eps,
                                        k_out=k_out, v_out=v_out)
        m = qkv.shape[0]
        q = torch.empty(m, self.nh, sp["hd"], dtype=torch.float16, device=qkv.device)
        _lib.call("sb_qkv_prep", qkv.data_ptr(), _F16, sp["nqkv"], L["q_norm"].data_ptr(), None, L["cos"].data_ptr(),
                  L["sin"].data_ptr(), pos.data_ptr(), 0, m, self.nh, sp["hd"], self.eps, q.data_ptr(), None, None, None,
                  None, None, self.dm.max_seq * sp["hd"], kern._stream())
        return q

    def _draw(self, out32, out16, at) -> None:
        """Next tokens from the last hidden rows: logits, softcap and sampling; then the step's bookkeeping."""
        dm = self.dm
        if self.B <= self.GEMV_ROWS:
            logits = torch.empty(self.B, self.vocab, device=dm.device)
            kern.lmhead_argmax(dm.lm_q, dm.lm_s, out32, logits=logits, want_tokens=False, bits=dm.lm_bits)
        else:  # f16: the GEMM's output type, steps of 2^-7 at logits of 8 to 16
            logits = kern.gemm_q4(out16, dm.lm_q, dm.lm_s, bits=dm.lm_bits,
                                  workspace=self._gemm_ws(self.B, (dm.lm_q,), self.H))
        kern.sample(logits, self.seeds, at, temperature=self.temperature, top_k=self.top_k, top_p=self.top_p,
                    min_p=self.min_p, softcap=self.softcap, tokens=self.tok)
        # -1 (every logit NaN or -inf) is no row of the embedding
        _lib.call("sb_step_advance", self.pos.data_ptr(), torch.clamp(self.tok, min=0).data_ptr(), self.cur.data_ptr(),
                  self.history.data_ptr(), self.dm.max_seq, self.B, kern._stream())

    # ------------------------------------------------------------------ prefill and decode
    def prefill(self, prompts, steps: int = 1) -> list[int]:
        """Run the batch's prompts packed through the layers, with pages for ``steps`` tokens
        more each; returns the first token drawn for each."""
        lens = [len(p) for p in prompts]
        if steps < 0:
            raise ValueError("steps must not be negative")
        if len(lens) != self.B or min(lens) < 1 or max(lens) + steps > self.dm.max_seq:
            raise ValueError(f"{self.B} prompts of 1 to {self.dm.max_seq - steps} tokens are wanted")
        dm, dev, T = self.dm, self.dm.device, sum(lens)
        tokens = torch.cat([torch.as_tensor(list(p), dtype=torch.int64) for p in prompts])
        rows = dm.embed_q.shape[0]
        if int(tokens.min()) < 0 or int(tokens.max()) >= rows:  # they are looked up without a check
            raise ValueError(f"tokens must lie in 0 .. {rows - 1}")
        with self._own_stream():
            left = self._reserve(lens, steps)
            host = torch.empty(3, T, dtype=torch.int32)
            host[0] = tokens
            host[1] = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens])
            host[2] = torch.repeat_interleave(torch.arange(self.B, dtype=torch.int32), torch.tensor(lens))
            tok, pos, seq = host.to(dev).unbind(0)
            ends = torch.tensor(lens, device=dev)
            plans, kv = {}, {}

            def attend(li, L, qkv):
                sp = L["spec"]
                if sp["own"]:
                    kv[li] = tuple(torch.empty(T, 1, sp["hd"], dtype=torch.float16, device=dev) for _ in range(2))
                k, v = kv[sp["src"] if not sp["own"] else li]
                q = self._append(li, L, qkv, pos, seq, k, v)
                key = (sp["hd"], sp["window"])
                if key not in plans:
                    plans[key] = kern.PackedPlan(lens, self.nh, 1, sp["hd"], window=sp["window"], device=dev)
                return kern.attn_prefill_packed(q, k, v, plans[key])

            x = torch.empty(T, self.H, device=dev)
            dm.embed(tok.data_ptr(), T, x.data_ptr(), None, kern._stream())
            out32, out16 = self._layers(x, T, attend)
            rows = torch.cumsum(ends, 0) - 1
            self.pos.copy_(ends - 1)
            self._draw(out32[rows], out16[rows], self.pos)
            first = self.tok.tolist()
        self.left = left
        return first

    def _step(self) -> None:
        """One token per sequence: cur at position pos."""
        x = torch.empty(self.B, self.H, device=self.dm.device)
        self.dm.embed(self.cur.data_ptr(), self.B, x.data_ptr(), None, kern._stream())

        def attend(li, L, qkv):
            sp = L["spec"]
            q = self._append(li, L, qkv, self.pos, None)
            return kern.attn_decode_paged(q, self.caches[li], self.table, self.pos, window=sp["window"],
                                          workspace=self.attn_ws[sp["hd"]])

        self._draw(*self._layers(x, self.B, attend), self.pos)

    def decode_step(self) -> None:
        """One step for the whole batch; captured as a CUDA graph on first use."""
        if self.left < 1:
            raise ValueError("the sequences outgrow max_seq or the pages that prefill reserved for them")
        with torch.cuda.stream(self.stream):
            if self.graph is None:
                saved = [t.clone() for t in (self.pos, self.cur, self.tok, self.history)]
                self._step()  # first calls set kernel attributes outside capture
                for t, was in zip((self.pos, self.cur, self.tok, self.history), saved):
                    t.copy_(was)
                torch.cuda.synchronize(self.dm.device)
                self.graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(self.graph, stream=self.stream):
                    self._step()
            self.graph.replay()
        self.left -= 1
        self.taken += 1

    def decode(self, steps: int) -> list[list[int]]:
        """``steps`` more tokens for every sequence (``prefill`` has to have reserved their pages)."""
        start = [n + self.taken for n in self.lens]
        if steps < 0 or steps > self.left:
            raise ValueError(f"there is room for {self.left} more steps (pages that prefill reserved, max_seq)")
        for _ in range(steps):
            self.decode_step()
        with torch.cuda.stream(self.stream):
            h = self.history.cpu()
        return [h[b, n:n + steps].tolist() for b, n in enumerate(start)]

    def generate(self, prompts, steps: int, **sampling) -> list[list[int]]:
        """``steps`` tokens (at least one) for each prompt with the given sampling settings (``set_sampling``)."""
        if steps < 1:
            raise ValueError("steps must be positive")
        self.set_sampling(**sampling)
        first = self.prefill(prompts, steps)
        rest = self.decode(steps - 1) if steps > 1 else [[] for _ in first]
        return [[t] + r for t, r in zip(first, rest)]
