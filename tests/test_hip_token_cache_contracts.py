"""Calls of the token cache and its attention that the contracts allow, at their edges: one sequence with many new tokens behind a long prefix, queries
in any order.  Plain forms: test_hip_token_cache.py."""
import pytest
import torch

from test_hip_token_cache import DEV, cache_case, cache_reference, near, ops, run_cache  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,Hq,Hkv,D,C,P,cap,alibi", [(150, 8, 2, 64, 170, 13000, 0.0, True), (131, 4, 1, 128, 131, 12000, 0.0, False), (33, 8, 1, 256, 700, 40000, 20.0, False),
                                                      (70, 16, 2, 96, 70, 15000, 0.0, True)])
def test_one_sequence_with_many_new_tokens_behind_a_long_prefix(ops, T, Hq, Hkv, D, C, P, cap, alibi, kind):  # noqa: F811
    g = torch.Generator().manual_seed(D)
    x = cache_case(g, 1, T, Hq, Hkv, D, C, P, "plain", kind)
    slopes = torch.exp2(-torch.arange(1, Hq + 1).float() * 8 / Hq) if alibi else None
    for n in (C, T - 3):                                                    # the second: three rows before the first token
        lens = torch.tensor([n], dtype=torch.int32)
        want, top, score = cache_reference(x, lens, "plain", D ** -0.5, cap, slopes, P)
        near(run_cache(ops, x, lens, "plain", D ** -0.5, cap, slopes, P), want, top, score, kind)


@pytest.mark.parametrize("B,T,Hq,Hkv,D,P", [(64, 2, 8, 2, 64, 30000), (1, 128, 8, 2, 64, 30000), (9, 16, 16, 1, 256, 5100)])
def test_the_order_of_the_queries_changes_no_bit_behind_a_long_prefix(ops, B, T, Hq, Hkv, D, P):  # noqa: F811
    g = torch.Generator().manual_seed(D)
    x = cache_case(g, B, T, Hq, Hkv, D, T + 20, P, "plain", torch.bfloat16)
    lens = torch.tensor([T + 20 - b % 20 for b in range(B)], dtype=torch.int32)
    want = run_cache(ops, x, lens, "plain", D ** -0.5, 0.0, None, P)
    q = x["q"].to(DEV)
    for view in (q.transpose(0, 1).contiguous().transpose(0, 1), q.transpose(1, 2).contiguous().transpose(1, 2), torch.cat((q, q), 1)[:, T:], torch.cat((q, q), -1)[..., :D]):
        assert torch.equal(view, q) and torch.equal(run_cache(ops, {**x, "q": view}, lens, "plain", D ** -0.5, 0.0, None, P), want)
