"""The written-out gradients of `attention_formula` are those of its output, by automatic differentiation of the same sums row by row."""
import math

import pytest
import torch

from attention_formula import formula, head_columns


@pytest.mark.parametrize("per_edge", [False, True])
@pytest.mark.parametrize("bias", [None, "edges", "table"])
def test_against_automatic_differentiation(per_edge, bias):
    gen = torch.Generator().manual_seed(0)
    irreps_qk, irreps_v, H, N, E = "4x0e+2x1o", "2x0e+2x1o", 2, 5, 17
    S = E if per_edge else 6
    new = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    t = {"q": new(N, 10), "k": new(S, 10), "v": new(S, 8), "g": new(N, 8), "rowptr": torch.tensor([2, 2, 5, 6, 14, 15]), "perm": torch.randperm(E, generator=gen),
         "src": None if per_edge else torch.randint(S, (E,), generator=gen), "bias": None, "buckets": None, "weight": 0.1 + torch.rand(E, generator=gen).double()}
    t["weight"][t["perm"][3]] = 0.0
    if bias == "table":
        t["bias"], t["buckets"] = new(4, H), torch.randint(4, (E,), generator=gen)
    elif bias == "edges":
        t["bias"] = new(E, H)
        t["bias"][t["perm"][7:9], 1] = -math.inf
    leaves = {n: t[n].clone().requires_grad_() for n in ("q", "k", "v", "bias", "weight") if t[n] is not None}
    cq, cv = head_columns(irreps_qk, H), head_columns(irreps_v, H)
    out = []
    for n in range(N):
        row = [torch.zeros(8, dtype=torch.float64)]
        for h in range(H):
            a, vs = [], []
            for s in range(t["rowptr"][n], t["rowptr"][n + 1]):
                e = t["perm"][s]
                r = e if per_edge else t["src"][e]
                if t["weight"][e] <= 0 or (bias == "edges" and t["bias"][e, h] == -math.inf):
                    continue
                b = 0.0 if bias is None else leaves["bias"][e, h] if bias == "edges" else leaves["bias"][t["buckets"][e], h]
                a.append((leaves["q"][n, cq[h]] * leaves["k"][r, cq[h]]).sum() / math.sqrt(cq.shape[1]) + b + leaves["weight"][e].log())
                vs.append(leaves["v"][r, cv[h]])
            if a:
                row.append(torch.zeros(8, dtype=torch.float64).index_add(0, cv[h], torch.softmax(torch.stack(a), 0) @ torch.stack(vs)))
        out.append(sum(row))
    out = torch.stack(out)
    want = {"out": out.detach(), **dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), t["g"])))}
    got = formula(irreps_qk, irreps_v, H, t, torch.float64)
    assert set(want) == set(got)
    for name, x in want.items():
        assert (got[name][0] - x).abs().max() < 1e-13 * (1 + x.abs().max()), name
