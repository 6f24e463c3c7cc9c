"""The paged cache beside the rest of the package, on the CPU: its custom ops'
schemas, fake implementations and refusals, copies of a table, the decode
benchmark's candidate, and the reference's import path."""
import copy
import importlib
import json
import pickle

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import kotflash_amd.ops  # noqa: F401  (registers the ops)
from kotflash_amd import benchmark_decode
from kotflash_amd.paged import PageTable


def test_schemas():
    ns = torch.ops.kotflash_amd
    assert str(ns.paged_decode.default._schema).endswith("bool causal, float scale) -> (Tensor, Tensor)")
    app = str(ns.paged_append_.default._schema)
    assert "Tensor(a0!) k_pages, Tensor(a1!) v_pages, Tensor new_k" in app and app.endswith("-> ()")
    res = str(ns.page_reserve_.default._schema)
    assert "Tensor(a0!) tables, Tensor(a1!) lengths, Tensor free_pages, Tensor(a3!) counters" in res
    trim = str(ns.page_trim_.default._schema)
    assert "Tensor(a2!) free_pages, Tensor(a3!) counters, Tensor new_lengths" in trim


def test_fakes():
    with FakeTensorMode():
        q = torch.empty(3, 8, 2, 64, dtype=torch.bfloat16)
        k = torch.empty(20, 2, 16, 64, dtype=torch.bfloat16)
        tables = torch.empty(3, 9, dtype=torch.int32)
        lengths = torch.empty(3, dtype=torch.int32)
        o, lse = torch.ops.kotflash_amd.paged_decode(q, k, k, tables, lengths, True, 0.125)
        assert o.shape == q.shape and o.dtype == q.dtype
        assert lse.shape == (3, 8, 2) and lse.dtype == torch.float32
        free, counters = torch.empty(20, dtype=torch.int32), torch.empty(4, dtype=torch.int32)
        slots = torch.ops.kotflash_amd.page_reserve_(tables, lengths, free, counters, lengths.clone(), 16, 7)
        assert slots.shape == (3, 7) and slots.dtype == torch.int64


def test_ops_refuse_host_tensors():
    t = PageTable(2, 64, num_pages=4, device="cpu")
    counts = torch.ones(2, dtype=torch.int32)
    state = (t.tables, t.lengths, t.free_pages, t.counters)
    with pytest.raises(RuntimeError, match="gfx950"):
        torch.ops.kotflash_amd.page_reserve_(*state, counts, 16, 1)
    with pytest.raises(RuntimeError, match="gfx950"):
        torch.ops.kotflash_amd.page_trim_(*state, counts, 16)
    k = torch.zeros(4, 1, 16, 8, dtype=torch.float16)
    new = torch.zeros(2, 1, 1, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU tensors"):
        torch.ops.kotflash_amd.paged_append_(k, k.clone(), new, new, torch.zeros(2, 1, dtype=torch.int64))
    with pytest.raises(ValueError, match="GPU tensors"):
        torch.ops.kotflash_amd.paged_decode(new, k, k, t.tables, t.lengths, False, 1.0)


@pytest.mark.parametrize("which,bad", [
    (0, lambda t: t[0]), (0, lambda t: t.t().contiguous().t()), (0, lambda t: t.long()), (1, lambda t: t[:1]),
    (2, lambda t: t[:0]), (2, lambda t: t[::2]), (3, lambda t: t[:2]), (3, lambda t: t.long()),
])
def test_ops_refuse_other_states(which, bad):
    t = PageTable(2, 64, num_pages=4, device="cpu")
    state = [t.tables, t.lengths, t.free_pages, t.counters]
    state[which] = bad(state[which])
    with pytest.raises(ValueError):
        torch.ops.kotflash_amd.page_reserve_(*state, torch.ones(2, dtype=torch.int32), 16, 1)


@pytest.mark.parametrize("again", [copy.deepcopy, lambda t: pickle.loads(pickle.dumps(t))])
def test_copies_are_tables_of_their_own(again):
    t = PageTable(2, 64, num_pages=4, device="cpu")
    t.reserve(17)
    c = again(t)
    c.trim(0)
    assert c.num_free() == 4 and int(c.free_count) == 4 and c.lengths.tolist() == [0, 0]
    assert t.num_free() == 0 and t.lengths.tolist() == [17, 17]
    c.reserve(torch.tensor([70, 1], dtype=torch.int32), width=70)
    assert int(c.refused) == 1 and int(t.refused) == 0


def test_benchmark_candidate(capsys):
    benchmark_decode.main(["--device", "cpu", "--batch", "2", "--q-heads", "4", "--kv-heads", "2", "--head-dim", "16",
                           "--kv-seq", "1030", "--page-size", "48", "--warmup", "1", "--iterations", "2",
                           "--repeats", "3"])
    report = json.loads(capsys.readouterr().out)
    assert set(report["results"]) == {"auto", "pytorch_expanded_sdpa", "preallocated_auto", "paged_auto"}
    for metric in ("attention_only", "append_plus_attention"):
        assert report["correctness"]["paged_auto"][metric]["within_tolerance"]
    with pytest.raises(SystemExit):
        benchmark_decode.parse_args(["--device", "cpu", "--page-size", "-1"])
    assert "--page-size" in capsys.readouterr().err


def test_reference_import_path():
    import kotflash

    assert importlib.import_module("kotflash.paged") is importlib.import_module("kotflash_amd.paged") is kotflash.paged


@pytest.mark.parametrize("how", ["auto", "fused", "hip"])
def test_a_step_traces_without_graph_breaks(how, monkeypatch):
    """Table, store and attention as the custom ops, in one graph. Nothing runs
    here: the kernels need a GPU."""
    from kotflash_amd import paged

    monkeypatch.setattr(paged, "_on_gfx950", lambda t: True)
    table = PageTable(2, 64, num_pages=8, device="cpu")
    cache = paged.PagedKVCache(table, 2, 64, dtype=torch.float16)
    most = torch.tensor([20, 40], dtype=torch.int32)

    class Traced(Exception):
        pass

    seen = []

    def backend(gm, inputs):
        seen.extend(str(n.target) for n in gm.graph.nodes if "kotflash_amd" in str(n.target))

        def run(*args):
            raise Traced
        return run

    def step(q, n):
        table.trim(most)
        return cache.append_and_attend(q, n, n, table.reserve(1), append_backend=how)

    torch._dynamo.reset()
    with pytest.raises(Traced):
        torch.compile(step, backend=backend, fullgraph=True)(torch.zeros(2, 4, 1, 64).half(),
                                                             torch.zeros(2, 2, 1, 64).half())
    assert [s.split(".")[1] for s in seen] == ["page_trim_", "page_reserve_", "paged_append_", "paged_decode"]
