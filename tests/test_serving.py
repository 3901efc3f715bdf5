"""The page bookkeeping of the serving example, without a GPU."""
import pytest

from npu_amd.serving import Pages


def test_pages_grow_by_need_and_are_given_back():
    p = Pages(pages=5, page=16, slots=2, max_pages=3)
    assert [at for at, _ in p.grow(0, 1)] == [0] and p.grow(0, 16) == []
    assert [at for at, _ in p.grow(0, 33)] == [1, 2]
    assert [at for at, _ in p.grow(1, 17)] == [0, 1]
    assert sorted(p.owned[0] + p.owned[1]) == list(range(5)) and not p.free
    with pytest.raises(RuntimeError, match="table holds 3"):
        p.grow(0, 49)
    with pytest.raises(RuntimeError, match="0 free pages, 1 are needed"):
        p.grow(1, 33)
    assert len(p.owned[1]) == 2
    p.release(0)
    assert len(p.free) == 3 and p.owned[0] == []
    assert [at for at, _ in p.grow(1, 48)] == [2]


@pytest.fixture
def server(monkeypatch):
    """A Server on the host, whose groups do nothing, and torch.cuda's graphs as stand-ins."""
    import contextlib

    import torch

    from npu_amd import serving

    class Stream:
        def wait_stream(self, other):
            pass

    class Graph:
        pass

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "current_stream", Stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "graph", lambda g: contextlib.nullcontext())
    monkeypatch.setattr(serving, "decoder_layer", lambda p, bufs, *a: bufs["out"])
    monkeypatch.setattr(serving.Server, "_draw", lambda self, x: self.tokens)
    return serving.Server(*serving.random_model(1, 64, 1, 64, 32, device="cpu"), n_heads=1, slots=2, pages=8, page=16,
                          max_pages=3)


def test_no_prefix_while_a_captured_step_lives(server):
    """A captured step holds the addresses of the step's buffers and the prefix's length."""
    graph, one = server.capture(), server.one
    with pytest.raises(RuntimeError, match="captured"):
        server.set_prefix([1, 2, 3])
    assert server.one is one and server.prefix_len == 0 and len(server.pages.free) == 8
    del graph
    server.set_prefix([1, 2, 3])
    assert server.prefix_len == 3 and server.one is not one


def test_room_is_made_for_all_sequences_or_none(server):
    """A full table, then no free page: nothing has changed, and the next attempt is the same."""
    state = lambda: (list(server.lens), list(server.pages.free), [list(p) for p in server.pages.owned],
                     server.page_table.tolist())
    server.add(0, [1] * 16), server.add(1, [1] * 48)
    server.prefill()
    before = state()
    for _ in range(3):
        with pytest.raises(RuntimeError, match="the table holds 3"):
            server.make_room()
        assert state() == before
    server.remove(1)
    server.add(1, [1] * 32)
    server.prefill()
    server.pages.free, rest = server.pages.free[:1], server.pages.free[1:]
    before = state()
    for _ in range(3):
        with pytest.raises(RuntimeError, match="1 free pages, 2 are needed"):
            server.make_room()
        assert state() == before
    server.pages.free += rest
    server.make_room()
    assert server.lens == [17, 33] and server.page_table[0, 1] >= 0 and server.page_table[1, 2] >= 0


def test_capture_leaves_what_the_last_step_gave(server, monkeypatch):
    """Tokens, their probabilities and the logits, for whoever reads them after capture()."""
    import torch

    def draw(self, x):
        self.logits += 1
        self.probs += 1
        return self.tokens.add_(1)

    monkeypatch.setattr(type(server), "_draw", draw)
    server.logits.zero_()
    server.add(0, [1, 2, 3])
    server.prefill()
    shown = lambda: [t.clone() for t in (server.kv_len, server.tokens, server.probs, server.logits)]
    before = shown()
    server.capture()
    assert all(map(torch.equal, shown(), before))


def test_prefill_takes_the_waiting_sequences_alone(server, monkeypatch):
    """A batch of the slots that have new tokens: the others would count as sequences where
    the attention chooses its tiles."""
    from npu_amd import serving
    ran = []
    monkeypatch.setattr(serving, "decoder_layer", lambda p, bufs, cache, batch, *a: ran.append((bufs, batch)) or bufs["out"])
    server.add(1, list(range(20)))
    server.prefill()
    (bufs, batch), = ran
    assert batch["q_start"].tolist() == [0, 20] and batch["kv_len"].tolist() == [20]
    assert batch["page_table"].tolist() == [server.page_table[1].tolist()] and bufs["Q"].shape[0] == 20
    server.remove(1)
    server.add(1, [4] * 3), server.add(0, [5, 6])
    server.prefill()
    _, batch = ran[1]
    assert batch["q_start"].tolist() == [0, 2, 5] and batch["kv_len"].tolist() == [2, 3]
    assert batch["page_table"].tolist() == server.page_table.tolist()
