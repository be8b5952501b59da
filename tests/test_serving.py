"""The serving operators together, as a user runs them: prompts into the paged
cache, token after token out of it, forks, windows, release and compaction --
each step against a forward of the whole sequence in 64 bits under the
harness's acceptance rule (|u - r| <= 0.002 or <= 0.02 |r|)."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import _tklib as tk
import optimized
from paged_cache import PagedCache

gpu = pytest.mark.gpu


def make_model(d=128, heads=4, ffn=256, layers=2, causal=True, seed=0):
    torch.manual_seed(seed)
    cfg = optimized.TransformerConfig(batch_size=1, seq_len=1, d_model=d, num_heads=heads, ffn_dim=ffn,
                                      num_layers=layers, causal=causal)
    return optimized.OptimizedTransformer(cfg).eval()


def stack(model, x, window=0, sinks=0):
    """The layer stack over one sequence [S, d] in 64 bits."""
    S, H, hd = x.shape[0], model.num_heads, model.head_dim
    i, j = torch.arange(S)[:, None], torch.arange(S)[None, :]
    seen = j <= i
    if window:
        seen = seen & ((i - j < window) | (j < sinks))
    seen = seen.to(x.device)
    w = lambda m: (m.weight.double(), m.bias.double())  # noqa: E731
    x = x.double()
    for layer in model.layers:
        a = layer.attention
        h = F.layer_norm(x, (x.shape[1],), *w(layer.norm1))
        q, k, v = (F.linear(h, *w(m)).view(S, H, hd).transpose(0, 1) for m in (a.q_proj, a.k_proj, a.v_proj))
        s = (q @ k.transpose(1, 2) * hd ** -0.5).masked_fill(~seen, -float("inf"))
        x = x + F.linear((torch.softmax(s, -1) @ v).transpose(0, 1).reshape(S, -1), *w(a.out_proj))
        h = F.layer_norm(x, (x.shape[1],), *w(layer.norm2))
        x = x + F.linear(F.gelu(F.linear(h, *w(layer.ffn_in))), *w(layer.ffn_out))
    return F.layer_norm(x, (x.shape[1],), *w(model.final_norm))


def agrees(got, want):
    err = (got.double() - want).abs()
    bad = (err > 0.002) & (err > 0.02 * want.abs())
    assert torch.isfinite(got).all() and not bool(bad.any()), f"{int(bad.sum())} off, worst {float(err.max()):.3g}"


def make_cache(model, max_seqs=8, num_pages=128, page_size=16, width=24):
    return PagedCache(num_layers=len(model.layers), num_pages=num_pages, page_size=page_size,
                      kv_heads=model.num_heads, head_dim=model.head_dim, max_seqs=max_seqs, max_pages_per_seq=width)


def test_serving_refuses_on_host():
    model = make_model(causal=False)
    with pytest.raises(tk.TKError, match="must be a CUDA tensor"):
        model.prefill(torch.zeros(1, 4, 128), None, [0])
    with pytest.raises(tk.TKError, match="must be a CUDA tensor"):
        model.decode_step(torch.zeros(1, 128), None, [0])
    with pytest.raises(ValueError, match="expected x"):
        model.decode_step(torch.zeros(1, 4, 128), None, [0])


@gpu
@pytest.mark.parametrize("d, heads", [(128, 4), (256, 4), (256, 2), (64, 8)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (24, 3)])
def test_prompt_then_tokens(cuda_device, d, heads, window, sinks):
    """Padded prompts, then 40 tokens each; every output agrees with the
    stack over the whole sequence so far."""
    model = make_model(d=d, heads=heads).cuda()
    lens, S, steps = [50, 1, 33, 64], 64, 40
    g = torch.Generator().manual_seed(1)
    seqs = [torch.randn(n + steps, d, generator=g).cuda() for n in lens]
    cache = make_cache(model)
    x = torch.zeros(4, S, d, device="cuda")
    mask = torch.zeros(4, S, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        x[b, :n], mask[b, :n] = seqs[b][:n], True
    slots = torch.tensor([5, 0, 3, 6], dtype=torch.int32, device="cuda")
    with torch.inference_mode():
        want = [stack(model, s, window, sinks) for s in seqs]
        out = model.prefill(x, cache, slots, mask, window=window, sinks=sinks)
        for b, n in enumerate(lens):
            agrees(out[b, :n], want[b][:n])
        for t in range(steps):
            out = model.decode_step(torch.stack([s[n + t] for s, n in zip(seqs, lens)]), cache, slots, window=window,
                                    sinks=sinks)
            agrees(out, torch.stack([w[n + t] for w, n in zip(want, lens)]))
    assert cache.seq_lens.tolist() == [lens[1] + steps, 0, 0, lens[2] + steps, 0, lens[0] + steps, lens[3] + steps, 0]
    cache.check()
    tk.check_device_errors(cuda_device)


@gpu
def test_forks_continue_on_their_own(cuda_device):
    """A prompt forked twice, the copies fed different tokens; then the first
    is released, the cache compacted and the others go on."""
    model = make_model(d=256, heads=4).cuda()
    g = torch.Generator().manual_seed(2)
    prompt = torch.randn(45, 256, generator=g).cuda()
    tails = torch.randn(3, 30, 256, generator=g).cuda()
    cache = make_cache(model)
    with torch.inference_mode():
        want = [stack(model, torch.cat([prompt, t])) for t in tails]
        cache.reserve([7], [100])  # another sequence's pages in the way, released later
        model.prefill(prompt[None], cache, [0])
        cache.fork([0, 0], [1, 2])
        for t in range(15):
            agrees(model.decode_step(tails[:, t], cache, [0, 1, 2]), torch.stack([w[45 + t] for w in want]))
        cache.release([7, 0])
        assert int(cache.compact()) == 2 + 2 * 2  # two shared full pages, two of their own each
        for t in range(15, 30):
            agrees(model.decode_step(tails[1:, t], cache, [1, 2]), torch.stack([w[45 + t] for w in want[1:]]))
    cache.check()


@gpu
def test_captured_step_serves_a_changing_batch(cuda_device):
    """One captured step for up to four rows; sequences come and go between
    replays, free rows are padding."""
    model = make_model(d=128, heads=4).cuda()
    g = torch.Generator().manual_seed(3)
    seqs = [torch.randn(60, 128, generator=g).cuda() for _ in range(3)]
    cache = make_cache(model, width=8)
    x, slots = torch.zeros(4, 128, device="cuda"), torch.full((4,), -1, dtype=torch.int32, device="cuda")
    with torch.inference_mode():
        want = [stack(model, s, 20, 2) for s in seqs]
        model.decode_step(x, cache, slots, window=20, sinks=2)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model.decode_step(x, cache, slots, window=20, sinks=2)
        at = {}
        for step in range(50):
            if step in (0, 5, 20):
                s = (0, 5, 20).index(step)
                model.prefill(seqs[s][None, :7 + s], cache, [s], window=20, sinks=2)
                at[s] = 7 + s
            if step == 35:
                cache.release([1])
                del at[1]
            rows = [-1, -1, -1, -1]
            for s in at:
                rows[(s + step) % 4] = s
                x[(s + step) % 4] = seqs[s][at[s]]
            slots.copy_(torch.tensor(rows, dtype=torch.int32))
            graph.replay()
            for s in at:
                agrees(out[(s + step) % 4], want[s][at[s]])
                at[s] += 1
            if max(at.values()) >= 59:
                break
    cache.check()


@gpu
def test_serving_refuses_on_device(cuda_device):
    model = make_model().cuda()
    cache = make_cache(model)
    x = torch.zeros(2, 4, 128, device="cuda")
    with pytest.raises(tk.TKError, match="causal"):
        make_model(causal=False).cuda().prefill(x, cache, [0, 1])
    with pytest.raises(ValueError, match="layers, heads"):
        make_model(layers=3).cuda().prefill(x, cache, [0, 1])
    for bad in (dict(window=-1), dict(sinks=-1)):
        with pytest.raises(ValueError):
            model.prefill(x, cache, [0, 1], **bad)
    with pytest.raises(ValueError):
        model.prefill(x[:, :0], cache, [0, 1])
    with pytest.raises(ValueError):
        model.prefill(x, cache, [0])
    model.prefill(x, cache, [0, 1])
    cache.check()
    model.prefill(x, cache, [1, 2])  # slot 1 holds a prompt already
    with pytest.raises(tk.TKError, match="has to be empty"):
        cache.check()
    with pytest.raises(tk.TKError):
        tk.check_device_errors(cuda_device)
    cache.reset()
    assert model.decode_step(x[:0, 0], cache, []).shape == (0, 128)
    cache.check()


def test_mask_lengths_follow_the_mask():
    """A mask tensor that is filled again is read again; one that is not keeps
    its lengths (no second look at the device)."""
    model = make_model()
    mask = torch.tensor([[1, 1, 0, 0], [1, 0, 0, 0]], dtype=torch.bool)
    first = model._prefix_lengths(mask)
    assert first.tolist() == [2, 1]
    assert model._prefix_lengths(mask) is first
    mask[0, 2] = True
    assert model._prefix_lengths(mask).tolist() == [3, 1]
    mask.fill_(True)
    assert model._prefix_lengths(mask) is None
    mask.copy_(torch.tensor([[1, 0, 0, 0], [0, 0, 0, 0]]))
    assert model._prefix_lengths(mask).tolist() == [1, 0]
    with torch.inference_mode():  # such tensors do not count their changes
        mask = torch.tensor([[1, 1, 0, 0]], dtype=torch.bool)
        assert model._prefix_lengths(mask).tolist() == [2]
        mask[0, 2] = True
        assert model._prefix_lengths(mask).tolist() == [3]


@gpu
def test_prefill_reads_a_mask_that_is_filled_again(cuda_device):
    """One mask buffer for every batch, refilled by torch operations and by a
    replayed graph: each prompt's own length reaches the cache and the output."""
    model = make_model(d=128, heads=4).cuda()
    g = torch.Generator().manual_seed(7)
    S = 24
    x = torch.randn(2, S, 128, generator=g).cuda()
    mask, fresh = (torch.zeros(2, S, dtype=torch.bool, device="cuda") for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mask.copy_(fresh)
    cache = make_cache(model)
    with torch.inference_mode():
        want = [stack(model, s) for s in x]
    for round_, lens in enumerate(([24, 5], [7, 24], [1, 2], [24, 24])):
        now = (torch.arange(S)[None, :] < torch.tensor(lens)[:, None]).cuda()
        if round_ % 2:
            fresh.copy_(now)
            graph.replay()
        else:
            mask.copy_(now)
        slots = [2 * round_, 2 * round_ + 1]
        with torch.no_grad():
            out = model.prefill(x, cache, slots, mask)
        assert cache.seq_lens[slots].tolist() == lens
        for b, n in enumerate(lens):
            agrees(out[b, :n], want[b][:n])
    cache.check()
    with pytest.raises(tk.TKError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            model.prefill(x, cache, [0, 1], mask)
    assert cache.seq_lens.tolist() == [24, 5, 7, 24, 1, 2, 24, 24]
    cache.check()


@gpu
def test_calls_refused_on_the_host_leave_the_books(cuda_device):
    """What a serving call raises for, it raises for before a token is
    reserved; a window beyond any sequence is none."""
    model = make_model().cuda()
    cache = make_cache(model)
    g = torch.Generator().manual_seed(9)
    x = torch.randn(2, 5, 128, generator=g).cuda()
    ones = torch.ones(2, 5, dtype=torch.bool, device="cuda")
    with torch.inference_mode():
        want = [stack(model, s) for s in x]
        out = model.prefill(x[:, :4], cache, [0, 1], window=2 ** 40)
        for b in range(2):
            agrees(out[b], want[b][:4])
        books = cache._books.clone()
        for error, call in (
            (ValueError, lambda: model.decode_step(x[:, 4], cache, [0, 1], max_len=-1)),
            (ValueError, lambda: model.decode_step(x[:, 4], cache, [0, 1], window=-1)),
            (TypeError, lambda: model.decode_step(x[:, 4], cache, [0, 1], window=8.0)),
            (TypeError, lambda: model.decode_step(x[:, 4], cache, [0, 1], max_len=8.0)),
            (ValueError, lambda: model.decode_step(x[:, 4], cache, [0, 1, 2])),
            (TypeError, lambda: model.prefill(x, cache, [2, 3], window=4, sinks=1.5)),
            (ValueError, lambda: model.prefill(x, cache, [2, 3], ones[:, :4])),
            (ValueError, lambda: model.prefill(x, cache, [2, 3], ones[:1])),
            (ValueError, lambda: model.prefill(x, cache, [2, 3, 4], ones)),
            (tk.TKError, lambda: model.prefill(x, cache, [2, 3], torch.tensor([[1, 0, 1, 0, 0]] * 2).cuda())),
        ):
            with pytest.raises(error):
                call()
            assert torch.equal(cache._books, books)
        out = model.decode_step(x[:, 4], cache, [0, 1], window=2 ** 40, sinks=2 ** 33, max_len=2 ** 62)
        agrees(out, torch.stack([w[4] for w in want]))
    cache.check()
