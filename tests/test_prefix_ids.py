"""Family ids of paged_prefix_attention in other types than int32: neighbours are of one family exactly if the ids that
the caller gave are equal."""
import importlib
import random

import pytest
import torch

pa = importlib.import_module("dsa_triton_ascend_amd.paged_attention")  # (the package has a function of that name)

BIG = [2 ** 40 + 1, 2 ** 40 + 1, 2 ** 40 + 2, 2 ** 40 + 2, 5, 5, -1, -2 ** 50, -2 ** 50, 2 ** 31, 2 ** 31 - 1, 2 ** 63 - 1,
       2 ** 63 - 1, 2 ** 32 + 5, 5]


def _links(ids):
    return [ids[i] >= 0 and ids[i] == ids[i - 1] for i in range(1, len(ids))]


def _check(given, ids):
    got = pa._groups(given, torch.device("cpu"))
    assert got.dtype is torch.int32 and got.is_contiguous() and got.numel() == len(ids)
    got = got.flatten().tolist()
    assert _links(got) == _links(ids)
    assert [x < 0 for x in got] == [x < 0 for x in ids]


def test_ids_past_32_bits():
    _check(torch.tensor(BIG), BIG)
    _check(torch.tensor(BIG)[None], BIG)
    _check(torch.tensor([[x, 0] for x in BIG])[:, 0], BIG)
    _check(BIG, BIG)
    _check(tuple(BIG[:1]), BIG[:1])
    _check(torch.tensor(BIG[:1]), BIG[:1])
    rng = random.Random(3)
    for _ in range(20):
        ids = [rng.choice([2 ** 33, 2 ** 33 + 1, 2 ** 34, -5, -2 ** 40, 7]) for _ in range(rng.randint(1, 200))]
        _check(torch.tensor(ids), ids)
        _check(ids, ids)


def test_unsigned_and_narrow_ids():
    ids = [2 ** 64 - 1, 2 ** 64 - 1, 2 ** 63, 3, 3, 2 ** 64 - 2]
    _check(torch.tensor([x - 2 ** 64 if x >= 2 ** 63 else x for x in ids]).view(torch.uint64), ids)
    _check(ids, ids)
    ids = [2 ** 32 - 1, 2 ** 32 - 1, 2 ** 31, 2 ** 31 + 1, 0, 0]
    _check(torch.tensor(ids).to(torch.uint32), ids)
    for t in (torch.int8, torch.int16, torch.int32, torch.uint8, torch.bool):
        ids = [0, 1, 1, 0, 0]
        _check(torch.tensor(ids).to(t), ids)
    assert pa._groups(torch.zeros(0, dtype=torch.int64), torch.device("cpu")).numel() == 0


def test_ids_that_are_no_integers_are_refused():
    import dsa_triton_ascend_amd as dsa
    bf = torch.bfloat16
    for ids in (torch.tensor([0.2, 0.7]), [0.2, 0.7], torch.zeros(2, dtype=torch.complex64)):
        with pytest.raises(ValueError, match="prefix_groups must be integers"):
            pa._groups(ids, torch.device("cpu"))
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm GPU device"):  # (before anything else of the device is looked at)
        dsa.paged_prefix_attention(torch.zeros(2, 1, 8, 128, dtype=bf), torch.zeros(4, 16, 2, 128, dtype=bf),
                                   torch.zeros(4, 16, 2, 128, dtype=bf), torch.zeros(2, 2, dtype=torch.int32), i,
                                   torch.tensor([2 ** 40, 2 ** 40]), i)


@pytest.mark.gpu
@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("least", [1, 2 ** 40])
def test_neighbouring_families_with_ids_past_32_bits(latent, least):
    import dsa_triton_ascend_amd as dsa
    from tests.test_prefix_attention_gpu import _compare, _make
    families = [(0, 96, [100, 150, 130]), (1, 96, [97, 120]), (2, 96, [160, 99, 98])]
    args, data, lens = _make(families, 1, 16, 1 if latent else 2, 128, 16, torch.bfloat16, latent, seed=2)
    args["min_tokens"] = least
    want = _compare(args, data, lens)
    ids = [2 ** 40 + 1] * 3 + [2 ** 40 + 2] * 2 + [2 ** 63 - 1] * 3
    for given in (torch.tensor(ids, device="cuda"), torch.tensor(ids), ids):
        for x, y in zip(dsa.paged_prefix_attention(**dict(args, prefix_groups=given)), want):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_captured_calls_with_ids_of_64_bits():
    import dsa_triton_ascend_amd as dsa
    from tests.test_prefix_attention_gpu import _compare, _make
    families = [(0, 96, [100, 150, 130]), (1, 96, [97, 120]), (2, 96, [160, 99, 98])]
    args, data, lens = _make(families, 1, 16, 2, 128, 16, torch.bfloat16, False, seed=2)
    whole = args["prefix_groups"].clone()
    args["prefix_groups"] = ids = torch.tensor([2 ** 40 + x for x in whole.tolist()], device="cuda")
    names = torch.tensor([[0, 1, 2], [7, 2 ** 50, 2 ** 31], [2 ** 33, 2 ** 34, 2 ** 35], [2 ** 62, 5, 2 ** 62]], device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        dsa.paged_prefix_attention(**args)
        with torch.cuda.graph(graph, stream=stream):
            out = dsa.paged_prefix_attention(**args)
    torch.cuda.synchronize()
    for name in names:
        ids.copy_(name[whole.long()])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _compare(args, data, lens, got=out)
        _compare(args, data, lens)
