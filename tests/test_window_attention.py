"""Sliding-window attention with first tokens that stay visible, against its
definition in 64 bits, and what it refuses.

Tolerance, per output element, for weights p_j = exp(s_j - max) and A = sum p_j
|v_j| / sum p_j: rounding each p_j to fp16 costs half a step, 2^-11 p_j (2^-25
below fp16's normal range); a quarter of the exponentials come from a cubic
with relative error 7.5e-5, in numerator and denominator; the fp32 scores are
off by at most (hd + 2) 2^-24 sum |q_i k_i| scale, which moves both by as much;
2^x and the rescaling add a few 2^-22; the output is rounded to fp16, 2^-11
|out| (2^-25 below its normal range)."""

from __future__ import annotations

import pytest
import torch

import _tklib as tk
import kernels

gpu = pytest.mark.gpu


def reference(q, k, v, scale, window, sinks, kv_len=None):
    """[B, S, H, hd] context and tolerance in 64 bits, one (b, h) at a time."""
    B, H, S, hd = q.shape
    G = H // k.shape[1]
    i = torch.arange(S, device=q.device)[:, None]
    j = torch.arange(S, device=q.device)[None, :]
    band = (j <= i) & ((i - j < window) | (j < sinks))
    out = torch.zeros(B, S, H, hd, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = S if kv_len is None else max(0, min(S, int(kv_len[b])))
        seen = band[:, :n]
        some = seen.any(1)
        for h in range(H):
            Q, K, V = q[b, h].double(), k[b, h // G, :n].double(), v[b, h // G, :n].double()
            s = (Q @ K.T * scale).masked_fill(~seen, -float("inf"))
            s_err = (hd + 2) * 2.0 ** -24 * scale * (Q.abs() @ K.abs().T).masked_fill(~seen, 0)
            s, s_err, rows = s[some], s_err[some].amax(1, keepdim=True) if n else s_err[some], some
            if s.shape[0] == 0:
                continue
            p = torch.exp(s - s.amax(1, keepdim=True))
            total = p.sum(1, keepdim=True)
            o = p @ V / total
            A = p @ V.abs() / total
            tiny = ((p < 2.0 ** -14) & (p > 0)).double() @ V.abs() / total * 2.0 ** -25
            out[b, rows, h] = o
            tol[b, rows, h] = (2.0 ** -11 + 2 * 7.5e-5 + 2 * s_err + 8 * 2.0 ** -22) * A + tiny + 2.0 ** -11 * o.abs() \
                + 2.0 ** -25
    return out, tol


def inputs(B, H, Hkv, S, hd, seed=0, scale_up=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(B, S, H + 2 * Hkv, hd, generator=g, device="cuda") * scale_up
    qkv = qkv.half().permute(0, 2, 1, 3)
    return qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]


def check(q, k, v, window, sinks, kv_len=None, scale=None, **kw):
    B, H, S, hd = q.shape
    scale = hd ** -0.5 if scale is None else scale
    got = kernels.window_attention(q, k, v, scale, window, sinks=sinks, kv_len=kv_len, **kw)
    tk.check_device_errors(q.device)
    assert got.shape == (B, S, H * hd) and got.dtype == torch.float16
    ref, tol = reference(q, k, v, scale, window, sinks, kv_len)
    err = (got.view(B, S, H, hd).double() - ref).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} off, first at {bad.nonzero()[0].tolist()}, worst " \
                                f"{float((err / tol.clamp(min=1e-30)).max()):.2f} x tolerance"
    return got


# ---------------------------------------------------------------------------
# refusals that need no device
# ---------------------------------------------------------------------------
def test_c_entry_refuses_on_host():
    lib = tk.lib()

    def call(q=16, k=16, out=16, qs=(64 * 512, 64, 512), ks=(64 * 128, 64, 128), ld=512, B=1, S=64, H=8, K=2, hd=64,
             scale=0.1, w=16, s=2):
        return lib.tk_attn_window(q, *qs, k, k, *ks, out, ld, B, S, H, K, hd, scale, w, s, None, None)

    for kw, status in ((dict(q=None), -1), (dict(out=None), -1), (dict(S=0), -1), (dict(K=3), -1), (dict(K=0), -1),
                       (dict(hd=96), -2), (dict(w=0), -1), (dict(s=-1), -1), (dict(scale=0.0), -1),
                       (dict(scale=float("inf")), -1), (dict(ld=504), -1), (dict(ld=516), -1), (dict(out=8), -1),
                       (dict(q=8), -1), (dict(qs=(64 * 512, 60, 512)), -1), (dict(ks=(0, 64, 128), B=2), -1),
                       (dict(qs=(64 * 512, 64, 64)), -2), (dict(S=2 ** 31), -2)):
        assert call(**kw) == status, kw
        assert lib.tk_last_error() != b""


def test_wrapper_refuses_on_host():
    q, k = torch.zeros(1, 4, 8, 64).half(), torch.zeros(1, 2, 8, 64).half()
    with pytest.raises(tk.TKError, match="no CPU fallback"):
        kernels.window_attention(q, k, k, 1.0, 4)
    with pytest.raises(tk.TKError, match="float16"):
        kernels.window_attention(q.float(), k.float(), k.float(), 1.0, 4)
    with pytest.raises(tk.TKError, match="strides"):
        kernels.window_attention(q, k, k.transpose(1, 2).contiguous().transpose(1, 2), 1.0, 4)
    for bad in ((q, k[:, :, :4], k[:, :, :4]), (q[:, :3], k, k), (q, k, k[:, :1]), (q[0], k, k), (q[:, :, :0], k, k)):
        with pytest.raises(ValueError):
            kernels.window_attention(*bad, 1.0, 4)


# ---------------------------------------------------------------------------
# values
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("hd", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("S, window, sinks", [(1, 1, 0), (100, 32, 4), (300, 64, 0), (700, 200, 130)])
def test_head_dims(cuda_device, hd, S, window, sinks):
    check(*inputs(2, 3, 3, S, hd, seed=S), window, sinks)


@gpu
@pytest.mark.parametrize("H, Hkv", [(4, 4), (4, 1), (6, 2), (16, 8)])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_head_layouts(cuda_device, H, Hkv, hd):
    check(*inputs(2, H, Hkv, 513, hd, seed=H), 150, 5)


@gpu
@pytest.mark.parametrize("S", [127, 128, 129, 255, 256, 257, 640, 1000])
@pytest.mark.parametrize("window", [1, 2, 127, 128, 129, 257, 100000])
def test_tile_edges(cuda_device, S, window):
    for hd, sinks in ((64, 0), (128, 3)):
        check(*inputs(1, 2, 1, S, hd, seed=S), window, sinks)


@gpu
@pytest.mark.parametrize("sinks", [0, 1, 127, 128, 129, 300, 5000])
@pytest.mark.parametrize("hd", [16, 64, 128, 256])
def test_first_tokens(cuda_device, sinks, hd):
    """First tokens that end inside, at and past a tile, before and inside the window."""
    check(*inputs(1, 2, 2, 1100, hd, seed=sinks), 140, sinks)


@gpu
@pytest.mark.parametrize("hd", [8, 32, 64, 128, 256])
@pytest.mark.parametrize("window, sinks", [(50, 0), (130, 4), (1000, 0)])
def test_padded_rows_and_rows_without_keys(cuda_device, hd, window, sinks):
    """kv_len per sequence; keys and values past it are NaN and infinite. Rows
    whose window holds no key are zero."""
    S, lens = 600, [600, 0, 1, 130, 128, 599, 300]
    q, k, v = inputs(len(lens), 2, 1, S, hd, seed=hd)
    for b, n in enumerate(lens):
        k[b, :, n:] = float("nan")
        v[b, :, n:] = float("inf")
    v[3, :, 140:] = float("nan")
    kv_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = check(q, k, v, window, sinks, kv_len)
    assert not got[1].any()
    if sinks == 0 and window == 50:
        assert not got[2, 50:].any() and not got[3, 180:].any()


@gpu
def test_lengths_out_of_range_are_clamped(cuda_device):
    q, k, v = inputs(3, 2, 2, 200, 64)
    lens = torch.tensor([-5, 200, 10 ** 6], dtype=torch.int32, device="cuda")
    check(q, k, v, 64, 2, lens)


@gpu
def test_wide_window_is_causal_attention(cuda_device):
    q, k, v = inputs(2, 4, 4, 900, 64)
    a = check(q, k, v, 900, 0)
    b = kernels.flash_attention(q, k, v, 64 ** -0.5, True)
    # the same products and exponentials in another order of tiles: two roundings apart at most
    torch.testing.assert_close(a.float(), b.float(), atol=2e-3, rtol=2.0 ** -9)


@gpu
def test_large_scores(cuda_device):
    """Scores of several hundred: the running maximum moves by more than the lazy rescale's margin."""
    for hd in (64, 128):
        check(*inputs(1, 2, 2, 600, hd, scale_up=5.0), 200, 8)


@gpu
def test_strides(cuda_device):
    """[B, H, S, hd] contiguous tensors, and q laid out unlike k and v."""
    q, k, v = inputs(2, 4, 2, 333, 64)
    a = check(q, k, v, 100, 4)
    assert torch.equal(a, check(q.contiguous(), k.contiguous(), v.contiguous(), 100, 4))
    assert torch.equal(a, check(q, k.contiguous(), v.contiguous(), 100, 4))
    wide = torch.full((2, 333, 4 * 64 + 40), 3.0, device="cuda").half()
    check(q, k, v, 100, 4, out=wide[:, :, :256])
    assert torch.equal(wide[:, :, :256], a) and bool((wide[:, :, 256:] == 3).all())
    one = inputs(1, 1, 1, 50, 32)
    check(*one, 7, 1)


@gpu
def test_long_prompt(cuda_device):
    """20,000 tokens: many items per CTA, ring and barrier phases run on."""
    check(*inputs(1, 4, 2, 20000, 64, seed=2), 1000, 64)
    check(*inputs(1, 2, 1, 12001, 128, seed=3), 300, 4)


@gpu
def test_many_padded_items_per_cta(cuda_device):
    g = torch.Generator().manual_seed(5)
    B, S = 48, 700
    lens = torch.randint(0, S + 1, (B,), generator=g).int().cuda()
    for hd in (32, 128):
        q, k, v = inputs(B, 8, 4, S, hd, seed=6)
        v[torch.arange(S, device="cuda")[None, :].expand(B, S).ge(lens[:, None].long())[:, None, :].expand(B, 4, S)] = \
            float("nan")
        check(q, k, v, 90, 3, lens)


@gpu
def test_repeats_bit_for_bit_and_replays(cuda_device):
    q, k, v = inputs(3, 8, 4, 1025, 128, seed=8)
    lens = torch.tensor([1025, 400, 77], dtype=torch.int32, device="cuda")
    out = torch.empty(3, 1025, 8 * 128, device="cuda").half()
    first = kernels.window_attention(q, k, v, 0.1, 256, 4, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.window_attention(q, k, v, 0.1, 256, 4, lens, out=out)
    for _ in range(5):
        out.fill_(7)
        graph.replay()
        assert torch.equal(out, first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = kernels.window_attention(q, k, v, 0.1, 256, 4, lens)
    torch.cuda.synchronize()
    assert torch.equal(second, first)


@gpu
@pytest.mark.parametrize("hd", [8, 64, 128, 256])
def test_one_head_with_its_rows_next_to_each_other(cuda_device, hd):
    """[B, 1, S, hd] contiguous keys and values, and a single query head: a
    token's row begins where the one before ends."""
    for B, H, S in ((1, 1, 130), (3, 4, 200), (2, 1, 1)):
        q, k, v = inputs(B, H, 1, S, hd, seed=S)
        got = check(q, k, v, 70, 2)
        assert torch.equal(got, check(q.contiguous(), k.contiguous(), v.contiguous(), 70, 2))


def one_entry_strides():
    """(k, v, whether their strides agree where they mean something)"""
    flat = torch.zeros(8192).half()
    view = lambda shape, strides: torch.as_strided(flat, shape, strides)  # noqa: E731
    return [(view((1, 2, 8, 64), (8192, 64, 128, 1)), view((1, 2, 8, 64), (3, 64, 128, 1)), True),
            (view((1, 1, 8, 64), (512, 512, 64, 1)), view((1, 1, 8, 64), (512, 7, 64, 1)), True),
            (view((2, 2, 1, 64), (128, 64, 128, 1)), view((2, 2, 1, 64), (128, 64, 9, 1)), True),
            (view((1, 2, 8, 64), (8192, 64, 128, 1)), view((1, 2, 8, 64), (8192, 512, 64, 1)), False)]


def test_strides_of_one_entry_are_not_compared():
    for k, v, same in one_entry_strides():
        q = torch.zeros(k.shape[0], 4, k.shape[2], 64).half()
        with pytest.raises(tk.TKError, match="no CPU fallback" if same else "identical strides"):
            kernels.window_attention(q, k, v, 1.0, 4)


@gpu
def test_strides_of_one_entry_may_differ(cuda_device):
    """k and v whose strides differ only where a dimension has one entry give
    what contiguous copies give."""
    g = torch.Generator(device="cuda").manual_seed(11)
    for k0, v0, same in one_entry_strides():
        if not same:
            continue
        k, v = (torch.as_strided(torch.randn(8192, generator=g, device="cuda").half(), t.shape, t.stride())
                for t in (k0, v0))
        q = torch.randn(k.shape[0], 4, k.shape[2], 64, generator=g, device="cuda").half()
        got = check(q, k, v, 4, 1)
        assert torch.equal(got, check(q, k.contiguous(), v.contiguous(), 4, 1))


@gpu
@pytest.mark.parametrize("window, sinks", [(2 ** 63 - 1, 0), (2 ** 63 - 1, 2 ** 63 - 1), (1, 2 ** 63 - 1), (2 ** 31, 2 ** 31)])
def test_windows_and_first_tokens_beyond_any_length(cuda_device, window, sinks):
    q, k, v = inputs(2, 2, 1, 300, 64)
    assert torch.equal(check(q, k, v, window, sinks), check(q, k, v, 300, 0))
