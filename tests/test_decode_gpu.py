"""A BlockStack answering token by token from paged caches: prefill, decode steps,
log probabilities of the picked tokens, with plain and with 4-bit weights,
against the whole forward pass over the same tokens.

f32: max-abs 1e-3, as the layer tests; bf16: 2 % relative L2 error, since every
intermediate is rounded to bf16 in both, at different places.
"""
import pytest
import torch

import haelixe_b200 as hx
from haelixe_b200 import _native as N

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
VOCAB, HIDDEN, HEADS, LAYERS = 211, 128, 2, 2


def _stack(dtype, causal=True):
    return hx.nn.BlockStack(VOCAB, HIDDEN, HEADS, LAYERS, device="cuda", dtype=dtype, causal=causal, init_std=0.05, seed=3)


def _near(got, want, dtype):
    got, want = got.float(), want.float()
    assert torch.isfinite(got).all()
    if dtype == F32:
        assert (got - want).abs().max() < 1e-3
    else:
        assert (got - want).norm() < 0.02 * want.norm()


def _generate(stack, prompts, lens, steps, slots):
    """Greedy tokens, their log probabilities and the logits of every step."""
    B = prompts.shape[0]
    columns = -(-(int(lens.max()) + steps) // slots)
    table = torch.randperm(B * columns, device="cuda").to(torch.int32).view(B, columns)
    caches = stack.caches(B * columns, slots, table)
    logits = stack.prefill(prompts, caches, lens)
    positions, tokens, logprobs, all_logits = lens.clone(), [], [], []
    for _ in range(steps):
        all_logits.append(logits)
        best = hx.nn.token_logprobs(logits, torch.zeros(B, dtype=torch.int32, device="cuda"), 1).top_ids[:, 0]
        logprobs.append(hx.nn.token_logprobs(logits, best).logprob)
        tokens.append(best)
        logits = stack.decode(best, caches, positions)
        positions += 1
    return torch.stack(tokens, 1), torch.stack(logprobs, 1), torch.stack(all_logits, 1)


def _check_against_whole_passes(stack, prompts, lens, out, dtype):
    tokens, logprobs, logits = out
    for b in range(prompts.shape[0]):
        n, steps = int(lens[b]), tokens.shape[1]
        ids = torch.cat([prompts[b, :n].long(), tokens[b].long()])[None]
        with torch.no_grad():
            want = stack(ids)[n - 1:n - 1 + steps]
        _near(logits[b], want, dtype)
        lp = torch.log_softmax(logits[b].double(), -1).gather(1, tokens[b].long()[:, None])[:, 0]
        assert (logprobs[b].double() - lp).abs().max() < 1e-5
        assert torch.equal(tokens[b].long(), logits[b].float().argmax(-1))


@pytest.mark.parametrize("dtype", [pytest.param(F32, id="f32"), pytest.param(BF16, id="bf16")])
@pytest.mark.parametrize("slots", [16, 5])
def test_generation_agrees_with_whole_passes(dtype, slots):
    stack = _stack(dtype)
    prompts = torch.randint(VOCAB, (3, 40), generator=torch.Generator().manual_seed(1)).cuda()
    lens = torch.tensor([40, 1, 23], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        out = _generate(stack, prompts, lens, 6, slots)
    _check_against_whole_passes(stack, prompts, lens, out, dtype)


@pytest.mark.parametrize("dtype", [pytest.param(F32, id="f32"), pytest.param(BF16, id="bf16")])
def test_generation_with_4_bit_weights(dtype):
    """Against the same stack with the weights that the 4 bits stand for."""
    stack, plain = _stack(dtype), _stack(dtype)
    for blk in plain.blocks:
        for part in (blk.mha.q_proj, blk.mha.k_proj, blk.mha.v_proj, blk.mha.out_proj, blk.mlp.linear1, blk.mlp.linear2):
            _through_4_bits(part)
    _through_4_bits(plain.head)
    stack.quantize_w4(32)
    prompts = torch.randint(VOCAB, (2, 17), generator=torch.Generator().manual_seed(2)).cuda()
    lens = torch.tensor([17, 9], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        out = _generate(stack, prompts, lens, 4, 8)
        _check_against_whole_passes(stack, prompts, lens, out, dtype)
        _near(stack(prompts), plain(prompts), dtype)
    assert sum(p.numel() for p in stack.blocks[0].mha.parameters()) == HIDDEN  # the norm's weight alone


def _through_4_bits(linear):
    packed, scales = hx.nn.quantize_w4(linear.weight, 32)
    q = torch.stack([(packed >> (4 * i)) & 15 for i in range(8)], 1).flatten(0, 1)
    w = (q - 8).float() * scales.float().repeat_interleave(32, 0)
    linear.weight = w.to(linear.weight.dtype)  # bf16: (q - 8) * scale rounds once


def test_a_sequence_left_out_keeps_its_cache():
    stack = _stack(BF16)
    prompts = torch.randint(VOCAB, (2, 12), generator=torch.Generator().manual_seed(4)).cuda()
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    caches = stack.caches(4, 16, table)
    logits = stack.prefill(prompts, caches)
    before = [(c.k[table[1].long()].clone(), c.v[table[1].long()].clone()) for c in caches]
    ids = logits.float().argmax(-1)
    stack.decode(ids, caches, torch.tensor([12, -1], dtype=torch.int32, device="cuda"))
    for c, (k, v) in zip(caches, before):
        assert torch.equal(c.k[table[1].long()], k) and torch.equal(c.v[table[1].long()], v)


def test_decode_step_in_a_graph():
    stack = _stack(BF16)
    prompts = torch.randint(VOCAB, (2, 12), generator=torch.Generator().manual_seed(5)).cuda()
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    eager, graphed = stack.caches(4, 16, table), stack.caches(4, 16, table)
    ids = stack.prefill(prompts, eager).float().argmax(-1)
    stack.prefill(prompts, graphed)
    at = torch.full((2,), 12, dtype=torch.int32, device="cuda")
    step_ids, step_at = ids.clone(), at.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        stack.decode(step_ids, graphed, step_at)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        logits = stack.decode(step_ids, graphed, step_at)
    for _ in range(3):
        want = stack.decode(ids, eager, at)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want)
        ids = want.float().argmax(-1)
        at += 1
        step_ids.copy_(ids)
        step_at += 1


def test_refusals():
    stack = _stack(BF16, causal=False)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        stack.prefill(torch.zeros(1, 4, dtype=torch.int64, device="cuda"), stack.caches(1, 16, table))
    stack = _stack(BF16)
    with pytest.raises(ValueError):
        stack.decode(torch.zeros(1, dtype=torch.int64, device="cuda"), stack.caches(1, 16, table)[:1],
                     torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError):  # 4-bit weights have no backward
        stack.quantize_w4(32).loss(torch.zeros(1, 4, dtype=torch.int64, device="cuda"),
                                   torch.zeros(4, dtype=torch.int64, device="cuda"))


class _Watched:
    """The library, with every call that launches work checked for the context's lock."""

    def __init__(self, lib, lock, seen):
        self._lib, self._lock, self._seen = lib, lock, seen

    def __getattr__(self, name):
        fn = getattr(self._lib, name)
        if name in _NO_LAUNCH:
            return fn

        def call(*args):
            self._seen[name] = self._seen.get(name, True) and self._lock.locked()
            return fn(*args)
        return call


_NO_LAUNCH = {"hx_last_error", "hx_status_string", "hx_paged_attention_workspace_size", "hx_sync", "hx_last_path"}


def test_every_call_holds_the_context_from_its_stream_to_its_launch(monkeypatch):
    """Otherwise a call in another thread could change the stream in between."""
    seen, lib = {}, N.lib()
    watched = _Watched(lib, hx.context().lock, seen)
    monkeypatch.setattr(N, "lib", lambda: watched)
    stack = _stack(BF16)
    ids = torch.randint(VOCAB, (2, 12), generator=torch.Generator().manual_seed(6)).cuda()
    stack.loss(ids, ids.reshape(-1)).backward()
    hx.optim.AdamW(1e-3).step([(p.detach(), p.grad) for p in stack.parameters()])
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    caches = stack.caches(4, 16, table)
    logits = stack.prefill(ids, caches)
    at = torch.full((2,), 12, dtype=torch.int32, device="cuda")
    stack.decode(ids[:, 0], caches, at)
    stack.quantize_w4(32).decode(ids[:, 0], caches, at)
    leaf = logits.detach().requires_grad_()
    hx.nn.token_logprobs(leaf, ids[:, 0]).logprob.sum().backward()
    x = torch.randn(2, 2, 64, 64, device="cuda", dtype=BF16)
    q, k = x.clone().requires_grad_(), x.clone()
    hx.flash_attention(q, k, x, 0.125, True).sum().backward()
    hx.flash_attention(q.detach().requires_grad_(), k, x, 0.125, True, rope_base=1e4).sum().backward()
    hx.rope_forward(x, 1e4), hx.rope_backward(x, 1e4), hx.attention.rope_forward_qk(x, k, 1e4)
    from haelixe_b200 import sharding

    sharding.reassemble_heads(x[None], torch.empty(2, 64, 2, 64, device="cuda", dtype=BF16), 1)
    assert len(seen) >= 20 and all(seen.values()), [n for n, held in seen.items() if not held]


@pytest.mark.parametrize("quantized", [False, True])
def test_two_threads_decode_on_streams_of_their_own(quantized):
    """Each with its own stack and caches: the logits of one after the other (cuBLAS may choose
    other products beside a second stream)."""
    import threading

    def job(seed, stream, out):
        (stack, ids, caches, at), logits = out["made"], []
        with torch.cuda.stream(stream):
            for i in range(12):
                logits.append(stack.decode((ids + i) % VOCAB, caches, at + i))
            stream.synchronize()
        out["logits"] = torch.stack(logits)

    def make(seed):
        stack = hx.nn.BlockStack(VOCAB, HIDDEN, HEADS, LAYERS, device="cuda", dtype=BF16, init_std=0.05, seed=seed)
        prompts = torch.randint(VOCAB, (2, 12), generator=torch.Generator().manual_seed(seed)).cuda()
        caches = stack.caches(4, 16, torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2))
        stack.prefill(prompts, caches)
        if quantized:
            stack.quantize_w4(32)
        return stack, prompts[:, 0], caches, torch.full((2,), 12, dtype=torch.int32, device="cuda")

    for turn in range(10):
        alone, both = [{"made": make(s)} for s in (7, 8)], [{"made": make(s)} for s in (7, 8)]
        torch.cuda.synchronize()
        for s in range(2):
            job(s, torch.cuda.Stream(), alone[s])
        threads = [threading.Thread(target=job, args=(s, torch.cuda.Stream(), both[s])) for s in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        for a, b in zip(alone, both):
            _near(b["logits"], a["logits"], BF16)


def test_layers_that_are_not_causal_do_not_answer_from_a_cache():
    """A whole pass of such a layer attends both ways, which neither a causal prompt nor a decode step does."""
    mha = _stack(BF16, causal=False).blocks[0]
    cache = _stack(BF16).caches(1, 16, torch.zeros(1, 1, dtype=torch.int32, device="cuda"))[0]
    x = torch.zeros(1, 4, HIDDEN, device="cuda", dtype=BF16)
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    seq, at = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")
    for layer in (mha, mha.mha):
        with torch.no_grad(), pytest.raises(ValueError):
            layer.prefill(x, cache, seq, at)
        with torch.no_grad(), pytest.raises(ValueError):
            layer.decode(x[:, 0], cache, one - 1, one - 1, one)
    assert not cache.k.any() and not cache.v.any()


def test_the_last_position_of_an_integer_is_outside_the_table():
    stack = _stack(BF16)
    caches = stack.caches(2, 16, torch.arange(2, dtype=torch.int32, device="cuda").view(2, 1))
    ids = torch.zeros(2, dtype=torch.int64, device="cuda")
    logits = stack.decode(ids, caches, torch.tensor([0, 2**31 - 1], dtype=torch.int32, device="cuda"))
    assert torch.isfinite(logits[0]).all() and torch.isnan(logits[1]).all()


def test_prompt_lengths_outside_the_prompt():
    """They give NaN logits, and the other prompts what they give alone."""
    stack = _stack(F32)
    ids = torch.randint(VOCAB, (6, 9), generator=torch.Generator().manual_seed(9)).cuda()
    table = torch.arange(6, dtype=torch.int32, device="cuda").view(6, 1)
    lens = torch.tensor([9, 0, 10, -1, 4, 2**31 - 1], dtype=torch.int32, device="cuda")
    for n in (lens, lens.long()):
        logits = stack.prefill(ids, stack.caches(6, 16, table), n)
        assert torch.isnan(logits[[1, 2, 3, 5]]).all()
        with torch.no_grad():
            _near(logits[0], stack(ids[:1])[8], F32)
            _near(logits[4], stack(ids[4:5])[3], F32)



def test_more_prompts_or_positions_than_the_table_holds_are_refused():
    stack = _stack(BF16)
    caches = stack.caches(4, 16, torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2))
    stack.prefill(torch.zeros(1, 32, dtype=torch.int64, device="cuda"), caches)
    before = [c.k.clone() for c in caches]
    with pytest.raises(ValueError):
        stack.prefill(torch.zeros(3, 4, dtype=torch.int64, device="cuda"), caches)
    with pytest.raises(ValueError):
        stack.prefill(torch.zeros(2, 33, dtype=torch.int64, device="cuda"), caches)
    for n in (1, 3):
        with pytest.raises(ValueError):
            stack.decode(torch.zeros(n, dtype=torch.int64, device="cuda"), caches,
                         torch.zeros(n, dtype=torch.int32, device="cuda"))
    assert all(torch.equal(c.k, k) for c, k in zip(caches, before))
    # A longer padded batch is fine when its lengths fit.
    lens = torch.tensor([32, 5], dtype=torch.int32, device="cuda")
    assert torch.isfinite(stack.prefill(torch.zeros(2, 40, dtype=torch.int64, device="cuda"), caches, lens)).all()
