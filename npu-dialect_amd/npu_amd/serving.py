"""Serving a Llama decoder from a paged cache: the layer's groups with the three
serving operators between them.

    s = Server(layers, embed, g_out, w_out, n_heads=8, slots=16, pages=1024)
    s.set_prefix(system_prompt)                  # once, shared by all sequences
    s.add(slot, prompt)                          # a new sequence's tokens
    s.prefill()                                  # -> their first drawn tokens
    s.step()                                     # a token for every sequence

A step launches, per layer, QKV, rotate and append, attention over the pages and the
three groups after it, then the head and the draw; nothing in it waits for the
device, so step() can be captured (capture()) and replayed while pages are
added to the table between replays.  ``python -m npu_amd.serving`` runs a small
random model.
"""
import weakref

import torch

from . import groups


def decoder_layer(p, bufs, cache, batch, n_heads, eps=1e-5, stream=None):
    """One decoder layer over a paged cache, as six groups.  ``p``: g1, g2, wq, wk,
    wv, wo, wg, wu, wd and the position tables cos_t, sin_t; ``bufs``: x, Q, K, V,
    A, h, act, out, ones, zeros, ws (caller-owned); ``cache``: (k_pages, v_pages);
    ``batch``: page_table, kv_len, q_start, prefix_table, prefix_len."""
    k_pages, v_pages = cache
    at = (batch["page_table"], batch["kv_len"])
    dh = k_pages.shape[3]
    # the rotation by position is the append's: here cos 1, sin 0 (Q and K are rounded to
    # bf16 by both, once more than where the QKV group rotates)
    groups.fused_llama_qkv_rope(bufs["x"], p["g1"], p["wq"], p["wk"], p["wv"], bufs["ones"], bufs["zeros"],
                                bufs["Q"], bufs["K"], bufs["V"], eps, stream)
    groups.fused_llama_rope_append(bufs["Q"], bufs["K"], bufs["V"], p["cos_t"], p["sin_t"], k_pages, v_pages, *at,
                                   bufs["Q"], q_start=batch["q_start"], prefix_len=batch["prefix_len"],
                                   stream=stream)
    groups.fused_llama_paged_attention(bufs["Q"], k_pages, v_pages, *at, bufs["A"], dh ** -0.5, bufs["ws"],
                                       q_start=batch["q_start"], prefix_table=batch["prefix_table"],
                                       prefix_len=batch["prefix_len"], stream=stream)
    groups.fused_llama_matmul_residual(bufs["A"], p["wo"], bufs["x"], bufs["h"], stream)
    groups.fused_llama_rmsnorm_swiglu(bufs["h"], p["g2"], p["wg"], p["wu"], bufs["act"], eps, stream)
    groups.fused_llama_matmul_residual(bufs["act"], p["wd"], bufs["h"], bufs["out"], stream)
    return bufs["out"]


class Pages:
    """Which pages of a cache are free, and whose the others are."""

    def __init__(self, pages, page, slots, max_pages):
        self.page, self.max_pages = page, max_pages
        self.free = list(range(pages - 1, -1, -1))
        self.owned = [[] for _ in range(slots)]

    def _check(self, n):
        if n > len(self.free):
            raise RuntimeError(f"the cache has {len(self.free)} free pages, {n} are needed")

    def take(self, n):
        self._check(n)
        return [self.free.pop() for _ in range(n)]

    def grow(self, slot, keys):
        """New pages of a slot for its first ``keys`` keys: [(place, page)]."""
        return [(at, page) for _, at, page in self.grow_all({slot: keys})]

    def grow_all(self, keys):
        """The same for several slots, {slot: keys}: [(slot, place, page)], or
        an error and no page for any of them."""
        new = {}
        for slot, n in keys.items():
            need = -(-n // self.page)
            if need > self.max_pages:
                raise RuntimeError(f"{n} keys need {need} pages, the table holds {self.max_pages}")
            new[slot] = max(0, need - len(self.owned[slot]))
        self._check(sum(new.values()))
        placed = []
        for slot, n in new.items():
            at = len(self.owned[slot])
            self.owned[slot].extend(self.take(n))
            placed += [(slot, at + i, page) for i, page in enumerate(self.owned[slot][at:])]
        return placed

    def release(self, slot):
        self.free.extend(reversed(self.owned[slot]))
        self.owned[slot] = []


class Server:
    """``layers``: decoder_layer's parameters without the position tables, bf16 [K, N]
    weights and f32 gains; embed bf16 [vocabulary, D]; w_out bf16 [D, vocabulary]."""

    def __init__(self, layers, embed, g_out, w_out, n_heads, slots, pages, page=64, max_pages=64, eps=1e-5,
                 theta=10000.0):
        dev, (self.V, self.D) = embed.device, embed.shape
        self.embed, self.g_out, self.w_out, self.H, self.eps = embed, g_out, w_out, n_heads, eps
        dh = self.D // n_heads
        self.slots, self.pages, self.F = slots, Pages(pages, page, slots, max_pages), layers[0]["wg"].shape[1]
        # positions count the prefix, which is itself a sequence of the table's width at most
        angle = torch.arange(2 * max_pages * page, device=dev, dtype=torch.float64)[:, None] * \
            theta ** (-torch.arange(0, dh, 2, device=dev, dtype=torch.float64) / dh)
        tables = {"cos_t": angle.cos().float(), "sin_t": angle.sin().float()}
        self.layers = [dict(p, **tables) for p in layers]
        cache = lambda: torch.empty((pages, n_heads, page, dh), dtype=torch.bfloat16, device=dev)
        self.cache = [(cache(), cache()) for _ in layers]
        ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)
        self.page_table, self.kv_len = ints(slots, max_pages) - 1, ints(slots)
        self.prefix_table, self.prefix_len = None, 0
        self.tokens, self.u = ints(slots), torch.zeros(slots, device=dev)
        self.probs = torch.zeros(slots, device=dev)
        self.settings = {"temperature": torch.ones(slots, device=dev), "top_k": ints(slots),
                         "top_p": torch.ones(slots, device=dev), "min_p": torch.zeros(slots, device=dev)}
        self.lens, self.waiting = [0] * slots, {}
        self.logits = torch.empty((slots, self.V), dtype=torch.bfloat16, device=dev)
        self.no_residual = torch.zeros_like(self.logits)
        self.sample_ws = groups.sample_workspace(self.logits)
        self.one = self._buffers(slots)
        self.graphs = weakref.WeakSet()  # captured steps: they hold one's addresses and prefix_len

    def _tokens(self, tokens):
        tokens = [int(t) for t in tokens]
        if not tokens or min(tokens) < 0 or max(tokens) >= self.V:
            raise ValueError(f"tokens have to be one or more of 0 .. {self.V - 1}")
        return tokens

    def _buffers(self, T, page_table=None):
        dev = self.embed.device
        e = lambda n: torch.empty((T, n), dtype=torch.bfloat16, device=dev)
        b = {n: e(self.D) for n in ("x", "Q", "K", "V", "A", "h", "out")}
        b["act"] = e(self.F)
        b["ones"] = torch.ones((T, self.D // self.H // 2), device=dev)
        b["zeros"] = torch.zeros_like(b["ones"])
        b["ws"] = groups.paged_attention_workspace(b["Q"], self.cache[0][0],
                                                   self.page_table if page_table is None else page_table,
                                                   self.prefix_len)
        return b

    def _run(self, bufs, tokens, batch):
        # (a row without a token is drawn as -1)
        torch.index_select(self.embed, 0, tokens.clamp(min=0), out=bufs["x"])
        for p, cache in zip(self.layers, self.cache):
            bufs["x"].copy_(decoder_layer(p, bufs, cache, batch, self.H, self.eps))
        return bufs["x"]

    def _draw(self, x):
        x = x.float()
        x = (x * (x.square().mean(1, keepdim=True) + self.eps).rsqrt() * self.g_out).to(torch.bfloat16)
        groups.fused_llama_matmul_residual(x, self.w_out, self.no_residual, self.logits)
        return groups.fused_sample_tokens(self.logits, self.u, self.tokens, self.sample_ws, probs=self.probs,
                                          **self.settings)

    def _place(self, keys):
        for slot, at, page in self.pages.grow_all(keys):
            self.page_table[slot, at] = page

    def set_prefix(self, tokens):
        """The keys and values of tokens that every sequence begins with, computed
        once; before any sequence is added and any step captured."""
        if self.prefix_len or any(self.lens) or self.waiting:
            raise RuntimeError("a prefix comes before all sequences")
        if self.graphs:
            raise RuntimeError("a prefix comes before capture(): a captured step goes on without it")
        tokens = self._tokens(tokens)
        dev, n = self.embed.device, len(tokens)
        if n > self.pages.max_pages * self.pages.page:
            raise ValueError(f"a prefix of {n} tokens, the table holds {self.pages.max_pages * self.pages.page}")
        own = self.pages.take(-(-n // self.pages.page))
        table = torch.tensor([own + [-1] * (self.pages.max_pages - len(own))], dtype=torch.int32, device=dev)
        lens = torch.tensor([n], dtype=torch.int32, device=dev)
        self._run(self._buffers(n, table), torch.tensor(tokens, device=dev),
                  {"page_table": table, "kv_len": lens, "q_start": torch.cat([lens * 0, lens]), "prefix_table": None,
                   "prefix_len": 0})
        self.prefix_table, self.prefix_len = table[0, :len(own)].contiguous(), n
        self.one = self._buffers(self.slots)

    def add(self, slot, tokens, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        """A sequence of these tokens (after the prefix) in a free slot."""
        if self.lens[slot] or slot in self.waiting:
            raise RuntimeError(f"slot {slot} is taken")
        tokens = self._tokens(tokens)
        self._place({slot: len(tokens)})
        self.waiting[slot] = tokens
        for name, value in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
            self.settings[name][slot] = value

    def remove(self, slot):
        self.waiting.pop(slot, None)
        self.pages.release(slot)
        self.lens[slot] = 0
        self.kv_len[slot] = 0
        self.page_table[slot] = -1

    def _batch(self, q_start=None, slots=None):
        """Of all slots, a token each, or of those that have new tokens."""
        of = lambda t: t if slots is None else t[slots]
        return {"page_table": of(self.page_table), "kv_len": of(self.kv_len), "q_start": q_start,
                "prefix_table": self.prefix_table, "prefix_len": self.prefix_len}

    def prefill(self):
        """The added sequences' tokens; draws each one's next (the other slots keep
        their tokens; their rows of probs and logits mean nothing until the next step)."""
        dev, new = self.embed.device, [self.waiting.get(s, []) for s in range(self.slots)]
        start = torch.tensor([0] + [len(t) for t in new], dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev)
        tokens = torch.tensor([t for ts in new for t in ts], dtype=torch.int64, device=dev)
        if not tokens.numel():
            raise RuntimeError("no sequence waits")
        drawn = self.tokens.clone()
        for s, t in self.waiting.items():
            self.lens[s] = len(t)
            self.kv_len[s] = len(t)
        # (a slot without new tokens would count as a sequence where tiles are chosen)
        slots = torch.tensor(sorted(self.waiting), device=dev)
        batch = self._batch(torch.cat([start[:1], start[slots + 1]]), slots)
        x = self._run(self._buffers(len(tokens), batch["page_table"]), tokens, batch)
        last = (start[1:].long() - 1).clamp(min=0)
        self._draw(x[last])
        fresh = (start[1:] > start[:-1])
        self.tokens.copy_(torch.where(fresh, self.tokens, drawn))
        self.waiting = {}
        return self.tokens

    def step(self):
        """A token a sequence, each slot's last one in (a free slot's row is
        computed and means nothing).  u: this step's random numbers."""
        self.make_room()
        return self._step()

    def make_room(self):
        """Pages for the next token of every sequence; the host's part of a step.
        Where a table or the cache is full it raises and changes nothing."""
        if self.waiting:
            raise RuntimeError("sequences wait for prefill()")
        self._place({s: n + 1 for s, n in enumerate(self.lens) if n})
        self.lens = [n + 1 if n else 0 for n in self.lens]

    def _step(self):
        self.kv_len.add_((self.kv_len > 0).int())
        return self._draw(self._run(self.one, self.tokens, self._batch()))

    def capture(self):
        """step() as a graph: make_room() before each replay().  The last step's
        tokens, probs and logits stay."""
        state = [(t, t.clone()) for t in (self.kv_len, self.tokens, self.probs, self.logits)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # once, uncaptured: the first call of a kernel asks for its occupancy
            self.kv_len.zero_()
            self._step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self._step()
        for t, was in state:
            t.copy_(was)
        graph.server = self  # what it reads and writes lives as long
        self.graphs.add(graph)
        return graph


def random_model(n_layers, D, H, F, V, seed=0, device="cuda"):
    """(layers, embed, g_out, w_out) of random weights."""
    g = torch.Generator().manual_seed(seed)
    w = lambda k, n: (torch.randn((k, n), generator=g) * k ** -0.5).to(torch.bfloat16).to(device)
    gain = lambda: torch.rand(D, generator=g).add_(0.5).to(device)
    layers = [{"g1": gain(), "g2": gain(), "wq": w(D, D), "wk": w(D, D), "wv": w(D, D), "wo": w(D, D), "wg": w(D, F),
               "wu": w(D, F), "wd": w(F, D)} for _ in range(n_layers)]
    embed = torch.randn((V, D), generator=g).to(torch.bfloat16).to(device)
    return layers, embed, gain(), w(D, V)


def main():
    g = torch.Generator().manual_seed(1)
    draw = lambda n: torch.randint(0, 4096, (n,), generator=g).tolist()
    s = Server(*random_model(4, 512, 8, 1408, 4096), n_heads=8, slots=8, pages=128)
    s.set_prefix(draw(100))
    for slot, n in enumerate((5, 40, 1, 130, 77)):
        s.add(slot, draw(n), temperature=0.8, top_k=50, top_p=0.95)
    s.u.copy_(torch.rand(8, generator=g))
    out = [s.prefill().tolist()]
    graph = s.capture()
    for _ in range(15):
        s.make_room()
        s.u.copy_(torch.rand(8, generator=g))
        graph.replay()
        out.append(s.tokens.tolist())
    for slot in range(5):
        print(f"sequence {slot}: {[row[slot] for row in out]}")


if __name__ == "__main__":
    main()
