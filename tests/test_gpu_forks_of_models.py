"""Forks of requests through every model that the engine serves: convolutions, state-space and other recurrent states, latents, and the tokens that a bigram table looks back at, go with the request."""
import copy
import importlib

import pytest
import torch

import lia_b200  # noqa: F401
from lia_b200.engine import Engine

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
MODELS = {"bebulorn": "Bebulorn", "bizetar": "Bizetar", "davasun": "Davasun", "pazivik": "Pazivik", "sekenex": "Sekenex", "zatusun": "Zatusun"}


def model(name, case, dtype):
    cases, module = importlib.import_module(f"{name}_cases"), importlib.import_module(f"lia_b200.modeling_{name}")
    cls = getattr(module, MODELS[name] + "ForCausalLM")
    return cls(getattr(module, MODELS[name] + "Config").from_dict(copy.deepcopy(cases.CASES[case])), "cuda", dtype).init_weights(3)


@pytest.mark.parametrize("name", MODELS)
@pytest.mark.parametrize("case,dtype", [("even", BF16), ("odd", F32), ("wide", BF16)], ids=["even", "odd", "wide"])
@pytest.mark.parametrize("graphs", [False, True])
def test_a_fork_goes_on_as_its_request_would(name, case, dtype, graphs):
    """Logits of forks are, bit by bit, those of requests that were never forked, token by token and in portions; the request goes on too, and a fork of a fork; what a fork does leaves the others alone."""
    m = model(name, case, dtype)
    g = torch.Generator().manual_seed(1)
    ids = lambda n: torch.randint(0, m.config.vocab, (n,), generator=g).tolist()  # noqa: E731
    text, ways = ids(41), [ids(12) for _ in range(4)]
    cut = lambda way: [way[:1], way[1:2], way[2:3], way[3:10], way[10:11], way[11:]]  # noqa: E731
    alone = []
    for way in ways:
        eng = Engine(m, 80, max_requests=6, graphs=graphs)
        eng.step([{"id": 0, "tokens": text}])
        alone.append([eng.step([{"id": 0, "tokens": t, "want": [len(t) - 1]}]) for t in cut(way)])
        assert all(torch.isfinite(x).all() for x in alone[-1])
    eng = Engine(m, 80, max_requests=6, graphs=graphs)
    for i in range(3):                                                       # slots that were others' before
        eng.step([{"id": f"gone {i}", "tokens": ids(30)}])
    eng.step([], end=["gone 1", "gone 2"])
    eng.step([{"id": "a", "tokens": text}])
    eng.fork("a", ["b", "c"])
    go = lambda rid, way, i: torch.equal(eng.step([{"id": rid, "tokens": cut(ways[way])[i], "want": [len(cut(ways[way])[i]) - 1]}]), alone[way][i])  # noqa: E731
    assert go("c", 2, 0)
    eng.fork("c", ["d"])
    for i in range(6):
        assert go("a", 0, i) and go("b", 1, i) and (i == 0 or (go("c", 2, i) and go("d", 2, i))), i
    eng.step([], end=["b"])
    eng.step([{"id": "e", "tokens": text}])
    eng.fork("e", ["f"])
    for i in range(6):
        assert go("f", 3, i), i
