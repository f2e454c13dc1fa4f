"""How many logits Engine.score_choices holds at a time: a stand-in for a model on the CPU, whose distribution after a token depends on all tokens before it."""
import pytest
import torch


class Model:
    device = torch.device("cpu")
    config = type("C", (), {"vocab": 11})
    rows = 0

    def new_state(self, n, cap):
        from lia_b200.seq_state import SlotState
        s = SlotState(n, cap, "cpu")
        s.sums = s.add_recurrent(())
        return s

    def forward_rows(self, ids, batch, want, slots, trace=None):
        self.rows += len(ids)
        out = []
        for t, (slot, _) in zip(ids.tolist(), batch.meta.tolist()):
            slots.sums[slot] = slots.sums[slot] * 0.5 + t
            out.append(self.logits(slots.sums[slot]))
        return None if want is None else torch.stack(out)[want.long()]

    def logits(self, x):
        return torch.sin(torch.arange(11.0) * (x + 2))


@pytest.fixture
def engine(monkeypatch):
    import __graft_entry__ as g
    g.build()
    from lia_b200 import ops
    from lia_b200.engine import Engine
    held = []

    def plain(logits, given, top=0):
        held.append(logits.shape[0])
        logp = torch.log_softmax(logits, -1)
        best, ids = logp.sort(dim=-1, descending=True, stable=True)
        return logp.gather(1, given.view(-1, 1))[:, 0], -(logp.exp() * logp).sum(-1), best[:, :top], ids[:, :top]
    monkeypatch.setattr(ops, "token_logprobs", plain)
    return lambda **kw: (Engine(Model(), 64, **kw), held)


@pytest.mark.parametrize("max_rows,steps", [(4096, 1), (115, 1), (114, 2), (16, 10), (3, 40)])
@pytest.mark.parametrize("prompt", [[8, 1, 5, 2], [6]])
def test_no_more_logits_than_a_pass_has_rows(engine, max_rows, steps, prompt):
    """Long answers go portion by portion, what fits a pass goes at once, and every number is what it is by the definition."""
    g = torch.Generator().manual_seed(2)
    choices = [torch.randint(0, 11, (n,), generator=g).tolist() for n in (40, 1, 33, 40, 1)]
    e, held = engine(max_requests=6, max_rows=max_rows)
    del held[:]
    got = e.score_choices(prompt, choices, top=2)
    assert max(held) <= max(max_rows, len(choices)) and sum(held) == 115 == e.model.rows - (len(prompt) - 1)
    assert len(held) <= steps and e.slots.live_tokens == 0
    for c, x in zip(choices, got):
        s, want, entropy = torch.zeros(()), [], []
        for t, nxt in zip(prompt + c[:-1], [None] * (len(prompt) - 1) + c):
            s = s * 0.5 + t
            if nxt is not None:
                logp = torch.log_softmax(e.model.logits(s), -1)
                want.append(float(logp[nxt]))
                entropy.append(float(-(logp.exp() * logp).sum()))
        assert x["logp"] == pytest.approx(want) and x["entropy"] == pytest.approx(entropy) and [len(a) for a in x["alternatives"]] == [2] * len(c)


def test_an_answer_that_does_not_fit_leaves_nothing_behind(engine):
    from lia_b200.seq_state import SlotError
    e, _ = engine(max_requests=3, max_rows=16)
    with pytest.raises(SlotError):
        e.score_choices([1, 2, 3], [[4] * 5, [5] * 70])
    assert e.slots.live_tokens == 0 and e.slots.owner == [None] * 3
