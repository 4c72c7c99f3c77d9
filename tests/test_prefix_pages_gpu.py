"""paged_prefix_attention where a prefix ends inside a page: whose page its last
tokens are in, sequence by sequence.  Against the softmax in 64 bits, with the
bounds of test_prefix_attention_gpu.py; rows of caches that nobody may read are NaN."""
import pytest
import torch

from tests.test_prefix_attention_gpu import _compare, _make

pytestmark = pytest.mark.gpu


def _name_pages(args, data, families, page, which, seed=0):
    """Rows that name the whole pages of the prefix themselves, of the members that ``which`` picks: the tokens of the
    page where it ends are their own, unlike the first's."""
    g = torch.Generator(device="cuda").manual_seed(seed + 100)
    table, latent = args["block_table"], args["value"] is None
    caches = [args["key"], args["key_rope"] if latent else args["value"]]
    hosted = table.tolist()
    b = 0
    for _, P, members in families:
        first, whole = b, P // page * page
        for i, n in enumerate(members):
            if i and which(i) and whole:
                table[b, :whole // page] = table[first, :whole // page]
                for x, y, c in zip(data[b], data[first], caches):
                    x[:min(whole, n)] = y[:min(whole, n)]  # (so far only members of a family have these)
                    end = min(P, n)
                    if end > whole:
                        x[whole:end] = torch.randn(end - whole, *x.shape[1:], generator=g, device="cuda").to(x.dtype)
                        c[hosted[b][whole // page], :end - whole] = x[whole:end]
            b += 1


CASES = [
    # N1, N2, D, S1, page, dtype, latent, families
    (8, 2, 128, 1, 16, "fp16", False, [(0, 650, [663, 697, 681, 673])]),
    (20, 4, 128, 2, 48, "bf16", False, [(0, 100, [140, 133, 102]), (-1, 50, [60, 70]), (1, 64, [66, 166, 90])]),
    (16, 1, 256, 1, 64, "fp16", False, [(0, 500, [999, 501, 640, 700]), (0, 130, [200, 300, 131])]),
    (8, 8, 64, 3, 7, "bf16", False, [(0, 33, [36, 40, 37, 60]), (2, 100, [130, 103, 200])]),
    (16, 1, 512, 2, 64, "fp16", True, [(0, 130, [132, 200, 141]), (1, 0, [50]), (2, 376, [400] * 9)]),
    (128, 1, 512, 1, 64, "bf16", True, [(0, 1001, [1003, 1300, 1100]), (1, 77, [78, 200])]),
    (9, 1, 256, 1, 16, "bf16", True, [(0, 300, [301, 330, 310])]),
    (3, 1, 128, 1, 3, "fp16", True, [(0, 31, [40, 33, 35]), (1, 64, [65, 64, 90])]),
]


@pytest.mark.parametrize("i", range(len(CASES)))
@pytest.mark.parametrize("members", ["all", "second", "none"])
@pytest.mark.parametrize("least", [1, 2 ** 40])
def test_prefix_ends_inside_a_page(i, members, least):
    """Together and sequence by sequence; rows that name the prefix's whole pages, and rows that name none or others."""
    N1, N2, D, S1, page, dtype, latent, families = CASES[i]
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype]
    args, data, lens = _make(families, S1, N1, N2, D, page, dtype, latent, seed=i)
    _name_pages(args, data, families, page, {"all": lambda j: True, "second": lambda j: j % 2, "none": lambda j: False}
                [members], i)
    _compare(dict(args, min_tokens=least), data, lens)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("least", [1, 2 ** 40])
@pytest.mark.parametrize("named", [False, True])
def test_rows_that_hold_zeros_for_the_prefix(latent, least, named):
    """Zeros are a page's id too, but not that of the prefix: such rows take all of it from the first's."""
    families = [(0, 75, [90 + i for i in range(70)])]
    args, data, lens = _make(families, 1, 4, 1, 128, 16, torch.bfloat16, latent, seed=3)
    table = args["block_table"]
    assert (table[1:, :4] == -1).all()
    assert int(table[0, 3]) != 0  # (the first's own page there is another one)
    table[1:, :4] = 0
    if named:
        table[1::2, :4] = table[0, :4]
        caches = [args["key"], args["key_rope"] if latent else args["value"]]
        for b in range(1, 70, 2):
            for x, c in zip(data[b], caches):
                x[64:75] = torch.randn(11, *x.shape[1:], device="cuda").to(x.dtype)
                c[int(table[b, 4]), :11] = x[64:75]
    _compare(dict(args, min_tokens=least), data, lens)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("least", [1, 2 ** 40])
def test_prefix_shorter_than_a_page(latent, least):
    """No whole page before its end: the first's page holds it."""
    families = [(0, 40, [50, 60, 45]), (1, 63, [64, 100])]
    args, data, lens = _make(families, 1, 8, 1 if latent else 2, 128, 64, torch.float16, latent, seed=5)
    _compare(dict(args, min_tokens=least), data, lens)


@pytest.mark.parametrize("latent", [False, True])
@pytest.mark.parametrize("shared", [64, 75])
@pytest.mark.parametrize("least", [1, 2 ** 40, None])
def test_is_paged_attention_of_a_forked_table(latent, shared, least):
    """Whole rows, as a plan or a fork leaves them: what each sequence's own row says, whatever length is given."""
    import dsa_triton_ascend_amd as dsa
    families = [(0, 64, [330, 400, 90]), (1, 64, [77, 300])]
    args, data, lens = _make(families, 1, 16, 1 if latent else 2, 512 if latent else 128, 16, torch.bfloat16, latent, seed=8)
    table = args["block_table"]
    table[1:3, :4], table[4, :4] = table[0, :4], table[3, :4]
    args["prefix_lengths"].fill_(shared)
    a = _compare(dict(args, min_tokens=least), data, lens)
    plain = {k: v for k, v in args.items() if not k.startswith("prefix") and k != "min_tokens"}
    b = dsa.paged_attention(**plain)
    for x, y in zip(a, b):
        assert torch.allclose(x.float(), y.float(), rtol=2.0 ** -6, atol=2.0 ** -6)
        assert least != 2 ** 40 or torch.equal(x, y)
