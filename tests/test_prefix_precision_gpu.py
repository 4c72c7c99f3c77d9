"""The grouped form of paged_prefix_attention keeps its weights as paged_attention does, as two values of the input type:
beyond the rounding of the output, its error is that of the scores and of sums in 32 bits.

Bound of an output o = sum w v, with m = sum w |v| and u = eps / 2 of the type:
  scores    in 32 bits, ds off at most (products of `cols` terms and the scale): a weight by 2 ds of itself
  weights   two values: 2^-16 of itself at most (bf16, 8 bits each); fp16 values end at 2^-24, so 2^-33 of the
            row's largest weight at most for each of 2^13 tokens: 2^-20
  sums      at most 2^8 additions one after the other in 32 bits (tiles of 32 tokens, then parts): 2^-16
  exp2      2^-20
so |err| <= (2 ds + 2^-14) m before the output is rounded, and u of the result more.  A weight rounded once adds u m.
"""
import pytest
import torch

from tests.test_prefix_attention_gpu import DTYPES, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N1,N2,D,S1,page,dtype,families", [
    (8, 2, 128, 1, 16, "bf16", [(0, 640, [663, 697, 681, 673])]), (64, 2, 128, 2, 64, "fp16", [(0, 4096, [4100, 4098, 4500])]),
    (64, 8, 128, 1, 48, "bf16", [(0, 3000, [3001 + i for i in range(9)]), (1, 96, [100, 97])]),
    (16, 4, 64, 1, 16, "bf16", [(0, 2048, [2049, 2100, 2050])]), (5, 1, 64, 3, 3, "fp16", [(0, 600, [603, 700])]),
    (16, 1, 256, 1, 64, "bf16", [(0, 1024, [1030, 1025, 1100])]), (40, 2, 256, 1, 16, "fp16", [(0, 960, [970, 990])]),
    (24, 1, 256, 2, 7, "bf16", [(0, 700, [702, 720, 777])])])
@pytest.mark.parametrize("least", [1, 2 ** 40])
def test_no_more_than_the_rounding_of_the_output(N1, N2, D, S1, page, dtype, families, least):
    import dsa_triton_ascend_amd as dsa
    args, data, lens = _make(families, S1, N1, N2, D, page, DTYPES[dtype], False, seed=7)
    out = dsa.paged_prefix_attention(**dict(args, min_tokens=least))[0].double()
    half, G = torch.finfo(DTYPES[dtype]).eps / 2, N1 // N2
    for b, n in enumerate(lens):
        for s in range(S1):
            k, v = (x[:n - S1 + 1 + s].double().transpose(0, 1).contiguous() for x in data[b])
            q = args["query"][b, s].double().view(N2, G, D)
            kt = k.transpose(1, 2).contiguous()
            w = torch.softmax(torch.matmul(q, kt) * args["scale_value"], -1)
            ds = (torch.matmul(q.abs(), kt.abs()) * args["scale_value"]).amax(-1, keepdim=True) * (D + 4) * 2.0 ** -24
            want, mag = torch.matmul(w, v), torch.matmul(w, v.abs())
            inner = mag * (2 * ds + 2.0 ** -14)
            tol = inner + (want.abs() + inner) * half + (2.0 ** -25 if dtype == "fp16" else 0)
            err = (out[b, s].view(N2, G, D) - want).abs()
            assert (err <= tol).all(), f"sequence {b}, token {s}: worst ratio {(err / tol).max():.3g}"
