"""Serving a Llama decoder from a paged cache: the layer's groups with the three
serving operators between them.

    s = Server(layers, embed, g_out, w_out, n_heads=8, slots=16, pages=1024)
    s.set_prefix(system_prompt)                  # once, shared by all sequences
    s.add(slot, prompt)                          # a new sequence's tokens
    s.prefill()                                  # -> their first drawn tokens
    s.step()                                     # a token for every sequence
    s.score(tokens)                              # the log probabilities of given tokens

A step launches, per layer, QKV, rotate and append, attention over the pages and the
three groups after it, then the head and the draw; nothing in it waits for the
device, so step() can be captured (capture()) and replayed while pages are
added to the table between replays.  With ``alternatives`` a step also leaves its
tokens' log probabilities and the best other tokens.

``Server(*quantize_model(layers, embed, g_out, w_out), ...)`` holds the weights in four
bits (e2m1 in blocks of 32) and takes activations in eight to the products.
``python -m npu_amd.serving [--mx]`` runs a small random model.
"""
import sys
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


def mx_weight(w):
    """A weight [K, N] as (e2m1 [N, K / 2], scales [N, K / 32]), for fused_mx_matmul."""
    k, n = w.shape
    q = torch.empty((n, k // 2), dtype=torch.uint8, device=w.device)
    return groups.fused_mx_quantize(w.t(), q, torch.empty((n, k // 32), dtype=torch.uint8, device=w.device))


def quantize_model(layers, embed, g_out, w_out):
    """The model with its weights in four bits: QKV's and the gate's and the other's side by
    side; gains and the embedding as they are."""
    side = lambda p, *names: mx_weight(torch.cat([p[n] for n in names], 1))
    return [{"g1": p["g1"], "g2": p["g2"], "wqkv": side(p, "wq", "wk", "wv"), "wo": side(p, "wo"),
             "wgu": side(p, "wg", "wu"), "wd": side(p, "wd")} for p in layers], embed, g_out, mx_weight(w_out)


def mx_decoder_layer(p, bufs, cache, batch, n_heads, eps=1e-5, stream=None, delta=None):
    """One decoder layer with weights of quantize_model: bufs["x"] becomes x + delta (what the
    layer before left, None: nothing) plus attention, and the rest of this layer's output, to be added
    to it, is returned.  ``bufs``: x, qkv, A, o, gu, d, q and s (e4m3 [T, D] and its scales),
    qf and sf ([T, F]), ws, mx_ws; the others as decoder_layer's."""
    k_pages, v_pages = cache
    at = (batch["page_table"], batch["kv_len"])
    x, qkv, gu, q, s, ws = (bufs[n] for n in ("x", "qkv", "gu", "q", "s", "mx_ws"))
    D, F, dh = x.shape[1], gu.shape[1] // 2, k_pages.shape[3]
    Q, K, V = qkv[:, :D], qkv[:, D:2 * D], qkv[:, 2 * D:]
    groups.fused_llama_add_rmsnorm(x, p["g1"], q, s, delta=delta, h=x, eps=eps, stream=stream)
    groups.fused_mx_matmul(q, s, *p["wqkv"], qkv, ws, stream)
    groups.fused_llama_rope_append(Q, K, V, p["cos_t"], p["sin_t"], k_pages, v_pages, *at, Q, q_start=batch["q_start"],
                                   prefix_len=batch["prefix_len"], stream=stream)
    groups.fused_llama_paged_attention(Q, k_pages, v_pages, *at, bufs["A"], dh ** -0.5, bufs["ws"],
                                       q_start=batch["q_start"], prefix_table=batch["prefix_table"],
                                       prefix_len=batch["prefix_len"], stream=stream)
    groups.fused_mx_quantize(bufs["A"], q, s, stream=stream)
    groups.fused_mx_matmul(q, s, *p["wo"], bufs["o"], ws, stream)
    groups.fused_llama_add_rmsnorm(x, p["g2"], q, s, delta=bufs["o"], h=x, eps=eps, stream=stream)
    groups.fused_mx_matmul(q, s, *p["wgu"], gu, ws, stream)
    groups.fused_mx_quantize(gu[:, F:], bufs["qf"], bufs["sf"], gate=gu[:, :F], stream=stream)
    return groups.fused_mx_matmul(bufs["qf"], bufs["sf"], *p["wd"], bufs["d"], ws, stream)


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
    weights and f32 gains; embed bf16 [vocabulary, D]; w_out bf16 [D, vocabulary]; or what
    quantize_model makes of them.  ``alternatives``: None, or how many other tokens (0: none) a
    step leaves beside its tokens' log probabilities: logprobs, entropy, ranks [slots],
    top_tokens, top_logprobs [slots, alternatives], of the whole softmax of its logits."""

    def __init__(self, layers, embed, g_out, w_out, n_heads, slots, pages, page=64, max_pages=64, eps=1e-5,
                 theta=10000.0, alternatives=None):
        dev, (self.V, self.D) = embed.device, embed.shape
        self.mx = "wqkv" in layers[0]
        self.embed, self.g_out, self.w_out, self.H, self.eps = embed, g_out, w_out, n_heads, eps
        dh = self.D // n_heads
        self.slots, self.pages = slots, Pages(pages, page, slots, max_pages)
        self.F = layers[0]["wgu"][0].shape[0] // 2 if self.mx else layers[0]["wg"].shape[1]
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
        self.sample_ws = groups.sample_workspace(self.logits)
        self.head = self._head_buffers(slots)
        self.answers = {}
        if alternatives is not None:
            f, k = (lambda *shape: torch.zeros(shape, device=dev)), alternatives
            self.answers = {"logprobs": f(slots), "entropy": f(slots), "ranks": ints(slots) - 1,
                            "top_tokens": ints(slots, k) - 1 if k else None, "top_logprobs": f(slots, k) if k else None}
            self.answers_ws = groups.token_logprobs_workspace(self.logits, k)
            for name, t in self.answers.items():
                setattr(self, name, t)
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
        if self.mx:
            b = {n: e(self.D) for n in ("x", "A", "o", "d")}
            b["qkv"], b["gu"] = e(3 * self.D), e(2 * self.F)
            b["q"], b["s"] = self._blocks(T, self.D)
            b["qf"], b["sf"] = self._blocks(T, self.F)
            p = self.layers[0]
            b["mx_ws"] = max((groups.mx_matmul_workspace(b[a], p[w][0]) for a, w in
                              (("q", "wqkv"), ("q", "wo"), ("q", "wgu"), ("qf", "wd"))), key=torch.numel)
        else:
            b = {n: e(self.D) for n in ("x", "Q", "K", "V", "A", "h", "out")}
            b["act"] = e(self.F)
            b["ones"] = torch.ones((T, self.D // self.H // 2), device=dev)
            b["zeros"] = torch.zeros_like(b["ones"])
        b["ws"] = groups.paged_attention_workspace(b["A"], self.cache[0][0],
                                                   self.page_table if page_table is None else page_table,
                                                   self.prefix_len)
        return b

    def _blocks(self, T, K):
        dev = self.embed.device
        return (torch.empty((T, K), dtype=torch.float8_e4m3fn, device=dev),
                torch.empty((T, K // 32), dtype=torch.uint8, device=dev))

    def _head_buffers(self, T):
        """What the head keeps for T rows."""
        if not self.mx:
            return {"no_residual": torch.zeros((T, self.V), dtype=torch.bfloat16, device=self.embed.device)}
        q, s = self._blocks(T, self.D)
        return {"q": q, "s": s, "ws": groups.mx_matmul_workspace(q, self.w_out[0])}

    def _run(self, bufs, tokens, batch):
        # (a row without a token is drawn as -1)
        torch.index_select(self.embed, 0, tokens.clamp(min=0), out=bufs["x"])
        if self.mx:
            delta = None
            for p, cache in zip(self.layers, self.cache):
                delta = mx_decoder_layer(p, bufs, cache, batch, self.H, self.eps, delta=delta)
            return bufs["x"].add_(delta)
        for p, cache in zip(self.layers, self.cache):
            bufs["x"].copy_(decoder_layer(p, bufs, cache, batch, self.H, self.eps))
        return bufs["x"]

    def _head(self, x, head, logits):
        if self.mx:
            groups.fused_llama_add_rmsnorm(x, self.g_out, head["q"], head["s"], eps=self.eps)
            return groups.fused_mx_matmul(head["q"], head["s"], *self.w_out, logits, head["ws"])
        x = x.float()
        x = (x * (x.square().mean(1, keepdim=True) + self.eps).rsqrt() * self.g_out).to(torch.bfloat16)
        return groups.fused_llama_matmul_residual(x, self.w_out, head["no_residual"], logits)

    def _draw(self, x):
        self._head(x, self.head, self.logits)
        groups.fused_sample_tokens(self.logits, self.u, self.tokens, self.sample_ws, probs=self.probs, **self.settings)
        if self.answers:
            groups.fused_token_logprobs(self.logits, self.tokens, workspace=self.answers_ws, **self.answers)
        return self.tokens

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

    def score(self, tokens, rows=128):
        """Of a sequence of tokens (after the prefix), without a slot: the log probability of
        each after the first, given those before it, and the entropy there, both
        [len - 1].  ``rows``: of logits at a time."""
        if rows < 1:
            raise ValueError(f"{rows} rows at a time")
        tokens = self._tokens(tokens)
        dev, n = self.embed.device, len(tokens)
        if n > self.pages.max_pages * self.pages.page:
            raise ValueError(f"{n} tokens, the table holds {self.pages.max_pages * self.pages.page}")
        own = self.pages.take(-(-n // self.pages.page))
        try:
            table = torch.tensor([own + [-1] * (self.pages.max_pages - len(own))], dtype=torch.int32, device=dev)
            lens, ids = torch.tensor([n], dtype=torch.int32, device=dev), torch.tensor(tokens, device=dev)
            x = self._run(self._buffers(n, table), ids, {
                "page_table": table, "kv_len": lens, "q_start": torch.cat([lens * 0, lens]),
                "prefix_table": self.prefix_table, "prefix_len": self.prefix_len})
            logprobs, entropy = torch.zeros(n - 1, device=dev), torch.zeros(n - 1, device=dev)
            following = ids[1:].to(torch.int32)
            for r0 in range(0, n - 1, rows):
                r1 = min(n - 1, r0 + rows)
                logits = torch.empty((r1 - r0, self.V), dtype=torch.bfloat16, device=dev)
                self._head(x[r0:r1], self._head_buffers(r1 - r0), logits)
                groups.fused_token_logprobs(logits, following[r0:r1], logprobs[r0:r1],
                                            groups.token_logprobs_workspace(logits), entropy=entropy[r0:r1])
        finally:
            # (later work that is given these pages comes behind on the stream)
            self.pages.free.extend(reversed(own))
        return logprobs, entropy

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
        their tokens; their rows of probs, logits and alternatives mean nothing until the next step)."""
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
        tokens, probs, logits and alternatives stay."""
        state = [(t, t.clone()) for t in (self.kv_len, self.tokens, self.probs, self.logits, *self.answers.values())
                 if t is not None]
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
    model = random_model(4, 512, 8, 1408, 4096)
    s = Server(*(quantize_model(*model) if "--mx" in sys.argv[1:] else model), n_heads=8, slots=8, pages=128,
               alternatives=3)
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
        print(f"sequence {slot}: {[row[slot] for row in out]}; the last at log p {s.logprobs[slot]:.2f}, "
              f"best {s.top_tokens[slot].tolist()}")
    logprobs, entropy = s.score([row[3] for row in out])
    print(f"sequence 3's tokens alone: log p {logprobs.mean():.2f}, entropy {entropy.mean():.2f} each")


if __name__ == "__main__":
    main()
