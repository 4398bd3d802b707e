"""The decoding operators have no derivatives: every way of differentiating through them raises, and what they store counts as a change (on meta tensors)."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

I32 = torch.int32


@pytest.fixture(scope="module", autouse=True)
def _ops():
    from multimodal_amd import _torch_ops

    _torch_ops.load()


def meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


def calls():
    """name -> (a function of one float tensor of the operator's, that tensor)."""
    ns = torch.ops.mmamd
    q, kv, pages, table, n = meta(3, 4, 64), meta(3, 2, 64), meta(9, 2, 16, 64), meta(3, 5, dtype=I32), meta(3, dtype=I32)
    refs, step, done = meta(9, dtype=I32), meta(2, 3, dtype=I32), meta(2, 3, dtype=torch.bool)
    return {
        "paged_attention of q": (lambda x: ns.paged_attention(x, pages, pages, table, n, None, None, None), q),
        "paged_attention of v": (lambda x: ns.paged_attention(q, pages, pages, table, n, kv, x, None), kv),
        "paged_attention of pages": (lambda x: ns.paged_attention(q, x, pages, table, n, None, None, None), pages),
        "paged_attention_into": (lambda x: (o := meta(3, 4, 64), ns.paged_attention_into(x, pages, pages, table, n, None, None, None, o))[0], q),
        "paged_append": (lambda x: (p := meta(9, 2, 16, 64), ns.paged_append(x, x, p, pages, table, n, None))[0], meta(3, 7, 2, 64)),
        "paged_fork": (lambda x: (ns.paged_fork(x, table, n, refs, n, None, 1), x * 1)[1], pages),
        "paged_compact": (lambda x: (ns.paged_compact(x, table, refs), x * 1)[1], pages),
        "beam_search_step of logits": (lambda x: ns.beam_search_step(x, meta(2, 3), step, done, None, 1, 0.0)[0], meta(6, 50)),
        "beam_search_step of scores": (lambda x: ns.beam_search_step(meta(6, 50), x, step, done, None, 1, 0.0)[0], meta(2, 3)),
    }


@pytest.mark.parametrize("name", list(calls()))
def test_every_kind_of_derivative_raises(name):
    call, x = calls()[name]
    with pytest.raises(RuntimeError, match="no gradient"):
        call(x.clone().requires_grad_())
    with torch.no_grad():
        assert not call(x.clone().requires_grad_()).requires_grad
    with fwad.dual_level(), pytest.raises(RuntimeError, match="no gradient"):
        call(fwad.make_dual(x.clone(), x.clone()))
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.func.grad(lambda t: call(t).sum())(x.clone())
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.func.jvp(call, (x.clone(),), (x.clone(),))
    call(x)  # and nothing else is refused
    with torch.inference_mode():
        call(x)


def test_what_is_stored_counts_as_a_change():
    """Autograd refuses a backward pass whose saved tensor was overwritten by one of these operators, as by any in-place operation."""
    ns = torch.ops.mmamd
    q, kv, table, n, refs = meta(3, 4, 64), meta(3, 2, 64), meta(3, 5, dtype=I32), meta(3, dtype=I32), meta(9, dtype=I32)
    for change in (lambda p: ns.paged_attention(q, p, p, table, n, kv, kv, None), lambda p: ns.paged_append(kv[:, None], kv[:, None], p, p, table, n, None),
                   lambda p: ns.paged_fork(p, table, n, refs, n, None, 1), lambda p: ns.paged_compact(p, table, refs),
                   lambda p: ns.paged_attention_into(p.view(-1)[:768].view(3, 4, 64), meta(9, 2, 16, 64), meta(9, 2, 16, 64), table, n, None, None, None, p.view(-1)[:768].view(3, 4, 64))):
        pages = meta(9, 2, 16, 64)
        w = meta(9, 2, 16, 64).requires_grad_()
        loss = (w * pages).sum()
        before = pages._version
        with torch.no_grad():
            change(pages)
        assert pages._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.no_grad():  # reading changes nothing
        pages = meta(9, 2, 16, 64)
        ns.paged_attention(q, pages, pages, table, n, None, None, None)
        assert pages._version == 0
    with torch.inference_mode():
        pages = meta(9, 2, 16, 64)
    ns.paged_append(kv[:, None], kv[:, None], pages, pages, table, n, None)  # a pool made for inference has no versions, and may still be used outside
