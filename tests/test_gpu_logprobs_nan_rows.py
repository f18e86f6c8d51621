"""GPU checks of starkv.token_logprobs on rows of many NaN: the alternatives are
theirs, by ascending index from the first on, as a stable descending sort has
them; more of them than a workgroup ranks at once, in one piece and in several."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("V,top", [(1, 1), (40, 40), (700, 3), (5000, 1), (5000, 64), (40000, 5), (131072, 20)])
def test_rows_of_nan(V, top, dtype):
    from starkv import token_logprobs
    g = torch.Generator().manual_seed(V)
    n = torch.randn(V, generator=g)
    at = torch.arange(V)
    rows = {"all": torch.full((V,), math.nan),
            "all but the first": torch.where(at == 0, n, math.nan),
            "the first": torch.where(at == 0, math.nan, n),
            "the first, the rest equal": torch.where(at == 0, math.nan, 1.5),
            "the first, the rest barred": torch.where(at == 0, math.nan, -math.inf),
            "every third": torch.where(at % 3 == 0, math.nan, n),
            "the first half": torch.where(at <= V // 2, math.nan, n),
            "negative NaN": torch.full((V,), -1, dtype=torch.int32).view(torch.float32)}
    x = torch.stack(list(rows.values())).to(dtype).cuda()
    want = torch.sort(x.float().cpu(), dim=-1, descending=True, stable=True).indices[:, :top]
    tok = torch.zeros(len(rows), dtype=torch.int64, device="cuda")
    res = token_logprobs(x, tok, top=top)
    torch.cuda.synchronize()
    bad = x.isnan().any(-1)
    for i, name in enumerate(rows):
        one = token_logprobs(x[i:i + 1], tok[i:i + 1], top=top)
        for how, ids in (("of many", res.top_ids[i]), ("alone", one.top_ids[0])):
            print(name, how, ids[:4].tolist(), flush=True)
            assert torch.equal(ids.cpu(), want[i]), (name, how)
        for r, j in ((res, i), (one, 0)):
            if bool(bad[i]):
                assert r.logprob[j].isnan() and r.entropy[j].isnan() and r.top_logprobs[j].isnan().all()
