"""Infinities and NaN among the tokens that count: what the definition makes of them."""
import math

import pytest
import torch

import test_shared_attention_gpu as A

pytestmark = pytest.mark.gpu

SETS = [(8, 2, 128, [([0, 1, 2, 3], 24)], [384 + 20, 384, 384 + 65, 384 + 200]),          # block units
        (8, 8, 64, [([0, 1], 24)], [384 + 40, 384 + 3]),                                  # units of single waves
        (32, 8, 128, [], [300, 17, 70])]                                                  # own pages alone


def definition(c):
    """out [B, Hq * D] in 64 bits."""
    Hq, Hkv, D = c["heads"]
    out = []
    for b, n in enumerate(c["lens"]):
        pages = c["table"][int(c["rows"][b]), : -(-n // 16)].long()
        k = c["k"][pages].double().permute(1, 0, 4, 2, 3, 5).reshape(Hkv, -1, D)[:, :n]
        v = c["v"][pages].double().permute(1, 0, 3, 2).reshape(Hkv, -1, D)[:, :n]
        s = (c["qkv"][b, :Hq].double().view(Hkv, Hq // Hkv, 1, D) * k[:, None]).sum(-1) / math.sqrt(D)
        w = torch.softmax(s, -1)
        out.append((w[..., None] * v[:, None]).sum(2).reshape(-1))
    return torch.stack(out)


@pytest.mark.parametrize("Hq,Hkv,D,groups,lens", SETS)
@pytest.mark.parametrize("pages", [(0, 1, 2, 3, 4), (6, 7), (0,)])
def test_scores_of_minus_infinity(ops, Hq, Hkv, D, groups, lens, pages):
    """Whole pages whose keys are -inf in a dimension in which every query is positive: their tokens have no weight.  Against the same tokens with
    keys far below the others, which have none either: the same bits."""
    print("case -inf", Hq, Hkv, D, pages, flush=True)
    c = A.build(ops, 3, groups, lens, Hq, Hkv, D, garbage=False)
    c["qkv"][:, :Hq, 0] = 4.0
    ids = torch.unique(c["table"][c["rows"].long()][:, list(pages)])
    ids = ids[ids >= 0].long()
    c["k"][ids, :, 0, 0, :, 0] = -60000.0                     # 4 x 60000 / 12: below the others by more than any weight shows
    want = A.call(ops, c)
    c["k"][ids, :, 0, 0, :, 0] = float("-inf")
    some = [b for b, n in enumerate(lens) if n > 16 * len(pages)]      # rows that have another token
    got = A.call(ops, c)
    assert bool(got[some].isfinite().all()) and torch.equal(got[some], want[some])
    assert bool(definition(c)[some].isfinite().all())


@pytest.mark.parametrize("Hq,Hkv,D,groups,lens", SETS)
@pytest.mark.parametrize("what", ["k", "v", "q"])
def test_nan_is_not_hidden(ops, Hq, Hkv, D, groups, lens, what):
    """NaN in a key, a value or a query that counts: NaN where the definition has it, and nowhere else."""
    print("case nan", Hq, Hkv, D, what, flush=True)
    c = A.build(ops, 4, groups, lens, Hq, Hkv, D, garbage=False)
    clean = A.call(ops, c)
    page = int(c["table"][int(c["rows"][0]), 5])
    if what == "q":
        c["qkv"][0, 1, 7] = float("nan")
    elif what == "k":
        c["k"][page, 1, 0, 1, 3, 2] = float("nan")
    else:
        c["v"][page, 1, 9, 3] = float("nan")
    got, want = A.call(ops, c), definition(c)
    assert bool(want.isnan().any()) and torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~got.isnan()], clean[~got.isnan()])
