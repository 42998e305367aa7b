"""Entries of some rows each that pass over a prefix together, beside the same entries by themselves, against
float64: the tolerance is masked attention's (test_masked_attention_gpu.py)."""
import pytest
import torch

from musc_hip._masked_attention_hip import Tokens, prefix_attention

from test_masked_attention_gpu import DTYPES, heads, i32, see as see_own
from test_prefix_attention_gpu import check_prefix, shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('b,t,p', [(300, 40, 300), (300, 40, 1500), (530, 33, 2000), (270, 70, 33), (100, 9, 1000), (40, 30, 5000)])
def test_many_entries(device, b, t, p, dtype):
    at = torch.arange(t)
    docs = torch.where(at[None] < (torch.arange(b) % (t + 1))[:, None], 0, -1)
    q, k, v = heads(device, dtype, b, t, t, 2, 2, 64)
    pk, pv = shared(device, dtype, p, 2, 64)
    side = Tokens(i32(docs, device), i32(at.expand(b, t).contiguous(), device))
    got = prefix_attention(q, k, v, pk, pv, 0.2, keys=side)
    some = torch.cat([torch.arange(0, b, 29), torch.tensor([b - 1])])
    check_prefix(got[some], q[some], k[some], v[some], pk, pv, 0.2, see_own(docs, docs, at, at)[some], docs[some] >= 0)
    assert (got.cpu()[docs < 0] == 0).all()
