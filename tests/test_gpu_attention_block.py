"""The attention's operators and the residual add in the modules that call them: the drop-in
FlashAttention module, the encoder block and the whole encoder in training, eager and
compiled."""
import pytest
import torch

import attention_reference as ref
from genet5_amd import attention
from genet5_amd.harness import encoder

pytestmark = pytest.mark.gpu

U = 2.0 ** -8


def rel(got, want):
    got, want = got.double(), want.double()
    return ((got - want).norm() / want.norm()).item()


OPTIONS = [dict(), dict(window_size=(40, 24), sink_tokens=3),
           dict(num_buckets=16, max_distance=50),
           dict(num_buckets=32, window_size=(60, 60), sink_tokens=2)]


@pytest.mark.parametrize("options", OPTIONS)
def test_self_attention_trains_like_the_torch_composition(cuda_device, options):
    """Output and every gradient of the HIP backend (bf16) against the PyTorch composition in
    fp32 from the same bf16 parameters, packed and batched.

    Bound: between input and any gradient lie at most 12 roundings to bf16 (q, k, v, P, out, o
    and their gradients, dS, the weight gradient), each at most U of its value: 12 U = 4.7e-2
    in the relative 2-norm if all were aligned."""
    torch.manual_seed(3)
    m = encoder.ALiBiSelfAttention(256, 4, **options).to(cuda_device)
    with torch.no_grad():
        for n, p in m.named_parameters():
            p.normal_(0, 1.0 if n == "relative_bias" else 0.08)
    m = m.to(torch.bfloat16)
    r = encoder.ALiBiSelfAttention(256, 4, backend="torch", **options).to(cuda_device)
    r.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    print(f"self attention {options}", flush=True)
    for shape, cu in (((2, 150, 256), None), ((1, 300, 256), torch.tensor([0, 90, 91, 300]))):
        h = torch.randn(*shape, device=cuda_device).to(torch.bfloat16)
        do = torch.randn(*shape, device=cuda_device).to(torch.bfloat16)
        hm, hr = h.clone().requires_grad_(True), h.float().requires_grad_(True)
        om, orr = m(hm, cu), r(hr, cu)
        gm = torch.autograd.grad(om, [hm, *m.parameters()], do)
        gr = torch.autograd.grad(orr, [hr, *r.parameters()], do.float())
        names = ["h"] + [n for n, _ in m.named_parameters()]
        for n, a, b in zip(["out"] + names, (om, *gm), (orr, *gr)):
            e = rel(a, b)
            print(f"  {n}: {e:.2e}", flush=True)
            assert e <= 12 * U, (n, e)


@pytest.mark.parametrize("kw", [dict(num_buckets=32), dict(window_size=(30, 30), sink_tokens=4),
                                dict(num_buckets=16, max_distance=40, window_size=(64, 0))])
def test_flash_attention_module(cuda_device, kw):
    """The drop-in module: its options reach the operator in inference and training, the
    fused projections are left out when only the bias needs a gradient, dropout follows
    torch.manual_seed and the mode."""
    torch.manual_seed(5)
    cfg = attention.FlashAttentionConfig(embed_dim=256, num_heads=4, num_kv_heads=2, dropout=0.2,
                                         **kw)
    m = attention.FlashAttention(cfg).to(cuda_device)
    if m.relative_bias is not None:
        with torch.no_grad():
            m.relative_bias.normal_()
        assert "relative_bias" in m.state_dict() and m.alibi_slopes(cuda_device) is None
    m = m.to(torch.bfloat16)
    h = torch.randn(2, 130, 256, device=cuda_device).to(torch.bfloat16)
    m.eval()
    with torch.no_grad():
        assert m._fused_projections(h)
        out, _ = m(h)
        q, k, v = (p(h).view(260, -1, 64) for p in (m.q, m.k, m.v))
    want = ref.attention(q, k, v, [0, 130, 260], 0.125, window=cfg.window_size,
                         sinks=cfg.sink_tokens, table=m.relative_bias,
                         slopes=m.alibi_slopes(cuda_device), max_distance=cfg.max_distance)
    want = want["out"].to(cuda_device).reshape(2, 130, 256) @ m.o.weight.double().t()
    assert rel(out, want) <= 6 * U          # q, k, v, P, the attention's output and o rounded
    if m.relative_bias is not None:
        m.requires_grad_(False)
        m.relative_bias.requires_grad_(True)
        assert not m._fused_projections(h)
        m(h)[0].float().pow(2).sum().backward()
        assert m.relative_bias.grad.abs().sum() > 0
        m.requires_grad_(True)
    m.train()
    outs = []
    for seed in (1, 1, 2):
        torch.manual_seed(seed)
        torch.cuda.manual_seed(seed)
        m.zero_grad()
        o, _ = m(h)
        o.float().pow(2).sum().backward()
        outs.append([o.detach()] + [p.grad.clone() for p in m.parameters()])
    for a, b in zip(outs[0], outs[1]):
        assert torch.equal(a, b)
    assert not torch.equal(outs[0][0], outs[2][0])
    assert all(torch.isfinite(g).all() for g in outs[0])


def test_encoder_trains_with_everything(cuda_device):
    """A step of the whole encoder, packed: window, sinks, learned bias and dropout in the
    attention, the experts and both residual adds; gradients for every parameter, the same
    for the same seed, and none of it in eval mode."""
    torch.manual_seed(7)
    m = encoder.GeneT5MoE(vocab_size=128, embed_dim=256, num_layers=2, num_heads=4, ff_dim=512,
                          num_experts=4, dropout=0.1,
                          attention_options=dict(window_size=(64, 64), sink_tokens=4,
                                                 num_buckets=32)).to(cuda_device)
    m = m.to(torch.bfloat16)
    ids = torch.randint(0, 128, (1, 500), device=cuda_device)
    cu = torch.tensor([0, 200, 201, 500])
    res = []
    for seed in (1, 1, 2):
        torch.manual_seed(seed)
        m.train()
        m.zero_grad(set_to_none=True)
        loss = m(ids, cu)["logits"].float().logsumexp(-1).mean()
        loss.backward()
        res.append([loss.detach()] + [p.grad for p in m.parameters()])
    names = [n for n, _ in m.named_parameters()]
    for n, g in zip(names, res[0][1:]):
        assert g is not None and torch.isfinite(g).all(), n
        assert g.abs().sum() > 0, n
    # the embedding's gradient is summed by torch's own kernel
    for n, a, b in zip(["loss"] + names, res[0], res[1]):
        assert torch.equal(a, b) or "embed" in n, n
    assert not torch.equal(res[0][0], res[2][0])
    m.eval()
    with torch.no_grad():
        a, b = m(ids, cu)["logits"], m(ids, cu)["logits"]
    assert torch.equal(a, b)


def test_dropout_probability_zero_is_the_block_without(cuda_device):
    """Training mode with dropout 0 and eval mode give the block's results as before."""
    torch.manual_seed(9)
    b = encoder.MoEEncoderBlock(256, 4, 512, 4).to(cuda_device).to(torch.bfloat16)
    h = torch.randn(1, 200, 256, device=cuda_device).to(torch.bfloat16)
    with torch.no_grad():
        want = b.eval()(h)
        assert torch.equal(b.train()(h), want)
        d = encoder.MoEEncoderBlock(256, 4, 512, 4, dropout=0.3).to(cuda_device).to(torch.bfloat16)
        d.load_state_dict(b.state_dict())
        assert torch.equal(d.eval()(h), want)
        assert not torch.equal(d.train()(h), want)


@pytest.mark.parametrize("kw", [dict(), dict(window_size=(20, 20), sink_tokens=2),
                                dict(table=16, dropout_p=0.2, dropout_seed=11)])
def test_compiled_equals_eager(cuda_device, kw):
    kw = dict(kw)
    T, H = 150, 4
    g = torch.Generator().manual_seed(13)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(cuda_device)
    n = kw.pop("table", None)
    leaves = [r(T, H, 64), r(T, 2, 64), r(T, 2, 64)] + ([r(n, H)] if n else [])
    do = r(T, H, 64)
    cu = torch.tensor([0, 40, 150], dtype=torch.int32, device=cuda_device)

    def f(q, k, v, *tab):
        return attention.flash_attn_varlen_func(q * 1, k, v, cu, cu, 110, 110,
                                                relative_bias=tab[0] if tab else None, **kw)

    res = []
    for fn in (f, torch.compile(f, fullgraph=True, backend="aot_eager")):
        x = [t.clone().requires_grad_(True) for t in leaves]
        out = fn(*x)
        res.append((out.detach(), *torch.autograd.grad(out, x, do)))
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_learned_bias_reaches_the_backward_of_the_table_only(cuda_device):
    """Only the table needs a gradient: the others get none, and the table's is the same as
    beside them."""
    T, H = 200, 4
    g = torch.Generator().manual_seed(17)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(cuda_device)
    q, k, v, do, tab = r(T, H, 64), r(T, H, 64), r(T, H, 64), r(T, H, 64), r(32, H)
    cu = torch.tensor([0, 200], dtype=torch.int32, device=cuda_device)
    tables = []
    for leaf in (False, True):
        x = [t.clone().requires_grad_(leaf) for t in (q, k, v)]
        t = tab.clone().requires_grad_(True)
        out = attention.flash_attn_varlen_func(*x, cu, cu, T, T, relative_bias=t)
        out.backward(do)
        assert all((p.grad is not None) == leaf for p in x)
        tables.append(t.grad)
    assert torch.equal(*tables)


def test_module_compiles_as_one_graph(cuda_device):
    """The module on a [B, L, D] batch, traced without a break, training and inference."""
    torch.manual_seed(19)
    cfg = attention.FlashAttentionConfig(embed_dim=256, num_heads=4, num_buckets=32,
                                         window_size=(50, 50), sink_tokens=2)
    m = attention.FlashAttention(cfg).to(cuda_device).to(torch.bfloat16)
    h = torch.randn(2, 120, 256, device=cuda_device).to(torch.bfloat16)
    f = torch.compile(lambda t: m(t)[0], fullgraph=True, backend="aot_eager")
    res = []
    for fn in (f, lambda t: m(t)[0]):
        m.zero_grad()
        x = h.clone().requires_grad_(True)
        out = fn(x)
        out.float().pow(2).sum().backward()
        res.append([out.detach(), x.grad] + [p.grad.clone() for p in m.parameters()])
    for a, b in zip(*res):
        assert torch.equal(a, b)
    with torch.no_grad():
        m.eval()
        m._fused_projections = lambda t: False
        assert torch.equal(f(h), m(h)[0])
