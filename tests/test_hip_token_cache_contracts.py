"""Calls of the token cache and its attention that the contracts allow, at their edges: one sequence with many new tokens behind a long prefix, queries
in any order, no keys at all, inputs that require gradients.  Plain forms: test_hip_token_cache.py."""
import pytest
import torch

from test_hip_token_cache import DEV, cache_case, cache_reference, masked_reference, near, ops, run_cache, run_masked, values  # noqa: F401

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


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Lq,Lk,Hq,Hkv,D,causal,alibi", [(5, 90000, 4, 1, 64, False, False), (3, 133000, 2, 1, 128, True, True), (2, 100011, 2, 2, 256, False, False)])
def test_a_row_of_more_than_64_parts(ops, Lq, Lk, Hq, Hkv, D, causal, alibi, kind):  # noqa: F811
    g = torch.Generator().manual_seed(D)
    q, k, v = torch.randn(1, Lq, Hq, D, generator=g).to(kind), values(g, 1, Lk, Hkv, D, kind=kind), values(g, 1, Lk, Hkv, D, kind=kind)
    slopes = torch.exp2(-6 - torch.arange(1, Hq + 1).float() * 8 / Hq) if alibi else None
    args = (D ** -0.5, causal, 0.0, slopes, torch.tensor([Lk - 1000], dtype=torch.int32), torch.tensor([Lk - Lq], dtype=torch.int32), None, None)
    want, top, score = masked_reference(q, k, v, *args)
    near(run_masked(ops, q, k, v, *args), want, top, score, kind)


def test_no_keys_at_all(ops):  # noqa: F811
    """Rows that see nothing are zero, with documents as without them."""
    z = lambda *s: torch.ones(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    for B, Lq in ((1, 1), (2, 5), (3, 700)):
        for causal in (True, False):
            for doc in (None, (i32(B, Lq), i32(B, 0))):
                out = ops.attention_masked(z(B, Lq, 4, 64), z(B, 0, 2, 64), z(B, 0, 2, 64), 1.0, causal, 0.0, None, i32(B), None, None, *(doc or (None, None)))
                assert out.shape == (B, Lq, 4, 64) and not out.any()
    with pytest.raises(RuntimeError, match="go together"):
        ops.attention_masked(z(2, 5, 4, 64), z(2, 0, 2, 64), z(2, 0, 2, 64), 1.0, True, 0.0, None, None, None, None, i32(2, 5), None)
    with pytest.raises(RuntimeError, match="k_doc must be"):
        ops.attention_masked(z(2, 5, 4, 64), z(2, 8, 2, 64), z(2, 8, 2, 64), 1.0, True, 0.0, None, None, None, None, i32(2, 5), i32(2, 0))


def test_inputs_that_require_gradients_are_refused(ops):  # noqa: F811
    """There is no backward pass: an answer without a gradient would be a gradient of zero to the caller."""
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=DEV)  # noqa: E731
    n = torch.ones(2, dtype=torch.int32, device=DEV)
    slopes = torch.ones(4, device=DEV)
    calls = {
        "cache_write": (lambda k, v: ops.cache_write(k, v, n, None, u8(2, 2, 8, 64), u8(2, 2, 8, 2), u8(2, 2, 8, 64), u8(2, 2, 8, 2), "mxfp8"), [z(2, 3, 2, 64), z(2, 3, 2, 64)]),
        "cache_attention": (lambda q, k, v, pk, pv, s: ops.cache_attention(q, k, v, None, None, n, pk, pv, None, None, "plain", 1.0, 0.0, s),
                            [z(2, 1, 4, 64), z(2, 2, 8, 64), z(2, 2, 8, 64), z(2, 5, 64), z(2, 5, 64), slopes]),
        "attention_masked": (lambda q, k, v, s: ops.attention_masked(q, k, v, 1.0, True, 0.0, s, None, None, None, None, None), [z(2, 5, 4, 64), z(2, 8, 2, 64), z(2, 8, 2, 64), slopes]),
    }
    for name, (call, inputs) in calls.items():
        call(*inputs)
        for i in range(len(inputs)):
            some = [t.clone().requires_grad_(j == i) for j, t in enumerate(inputs)]
            with pytest.raises(RuntimeError, match=f"{name} has no backward pass"):
                call(*some)
            with torch.no_grad():
                call(*some)
            with torch.inference_mode():
                call(*some)
            call(*(t.detach() for t in some))
