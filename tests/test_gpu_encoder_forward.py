"""GPU: what the packed encoder computes in, keeps and refuses — under autocast, without gradients, in train mode."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
transformers = pytest.importorskip("transformers")


def bert(layers=2, hidden=64, heads=2, dropout=0.0, seed=3):
    torch.manual_seed(seed)
    cfg = transformers.BertConfig(vocab_size=200, hidden_size=hidden, num_hidden_layers=layers, num_attention_heads=heads,
                                  intermediate_size=2 * hidden, max_position_embeddings=64, attn_implementation="eager",
                                  hidden_dropout_prob=dropout, attention_probs_dropout_prob=dropout)
    m = transformers.BertModel(cfg).eval()
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(2.0).add_(torch.randn(p.shape) * 0.02)
    return m.cuda()


def texts(B=7, S=31, seed=0):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(1, S + 1, (B,), generator=g)
    return torch.randint(0, 200, (B, S), generator=g).cuda(), (torch.arange(S)[None] < lens[:, None]).long().cuda()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_rows_between_the_products_stay_float32_under_autocast(dt):
    """Products that add nothing: what is left are the embeddings, the residual sums and the norms, which autocast runs in
    float32 — with them the result is the float32 one, whatever type the products take."""
    from two_towers_overlords_amd.encoder import PackedBertEncoder

    m = bert()
    with torch.no_grad():
        for layer in m.encoder.layer:
            for d in (layer.attention.output.dense, layer.output.dense):
                d.weight.zero_()
                d.bias.zero_()
    ids, mask = texts()
    with torch.no_grad():
        want = PackedBertEncoder(m).padded(ids, mask)
        with torch.autocast("cuda", dtype=dt):
            got = PackedBertEncoder(m).padded(ids, mask)
            stock = m(input_ids=ids, attention_mask=mask)[0] * mask.unsqueeze(-1)
    assert stock.dtype == torch.float32
    assert torch.equal(got, want)  # the same float32 operations on the same values
    # five norms of 64 terms: a mean and a variance of at most 2 (64 + 8) roundings each, on values of at most 8
    assert float((got - stock).abs().max()) <= 5 * 2 * (64 + 8) * 2.0 ** -24 * 8


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_autocast_is_as_close_to_64_bits_as_the_stock_forward(dt):
    """Both round the operands and results of the same products to the type; the packed forward rounds nothing else (it keeps
    more: activations and probabilities are formed in fp32).  The two errors are sums of as many roundings of random sign, so
    their root mean squares over some ten thousand values differ by little: a quarter is allowed."""
    from two_towers_overlords_amd.encoder import PackedBertEncoder

    m = bert(layers=4)
    ids, mask = texts(B=40)
    on = mask.bool()
    with torch.no_grad():
        want = copy.deepcopy(m).double()(input_ids=ids, attention_mask=mask)[0][on]
        with torch.autocast("cuda", dtype=dt):
            got = PackedBertEncoder(m).padded(ids, mask)[on]
            stock = m(input_ids=ids, attention_mask=mask)[0][on]
    rms = lambda t: float((t.double() - want).pow(2).mean().sqrt())
    assert rms(got) <= 1.25 * rms(stock), (rms(got), rms(stock))


def test_gradients_reach_every_weight_under_autocast():
    from two_towers_overlords_amd.encoder import PackedBertEncoder

    m = bert()
    ids, mask = texts()
    up = torch.randn(*ids.shape, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * mask.unsqueeze(-1)
    grads = {}
    for name, f in (("packed", lambda: PackedBertEncoder(m).padded(ids, mask)), ("stock", lambda: m(input_ids=ids, attention_mask=mask)[0])):
        m.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out = f()
        (out * up).sum().backward()
        grads[name] = {n: p.grad.double() for n, p in m.named_parameters() if p.grad is not None and bool(p.grad.any())}
    ref = copy.deepcopy(m).double()
    ref.zero_grad()
    (ref(input_ids=ids, attention_mask=mask)[0] * up.double()).sum().backward()
    want = {n: p.grad for n, p in ref.named_parameters() if p.grad is not None and bool(p.grad.any())}
    top = max(float(w.norm()) for w in want.values())
    assert len(want) >= 30
    for n, w in want.items():
        if float(w.norm()) < 1e-6 * top:  # key biases: their gradient is zero but for rounding
            continue
        err = float((grads["packed"][n] - w).norm())
        # a chain of 2 layers x 8 products either way, each rounded to 2^-9 of its size
        assert err <= 2 * 2 * 8 * 2.0 ** -9 * max(float(w.norm()), 1e-2 * top), (n, err, float(w.norm()))


def two_towers(m, **kw):
    from two_towers_overlords_amd.model import TwoTowersModel

    return TwoTowersModel(projection_dim=16, tokenizer=lambda *a, **k: None, pretrained_model=m, encoder_mode="bert", encoder_impl="hip", **kw).cuda()


def test_a_frozen_encoder_with_dropout_runs_in_train_mode():
    """train_epoch_optimized switches the model to train mode by itself; the frozen encoder's features are eval mode's."""
    from two_towers_overlords_amd.model import TripletLoss
    from two_towers_overlords_amd.training import train_epoch_optimized

    model = two_towers(bert(dropout=0.1))
    ids, mask = texts()
    want = model.query_tower.pool_tokens({"input_ids": ids, "attention_mask": mask})
    opt = torch.optim.Adam([p for p in model.parameters() if p.requires_grad], lr=1e-3)
    batches = [tuple(texts(B=6, S=20, seed=10 * i + r) for r in range(3)) for i in range(2)]
    avg = train_epoch_optimized(model, batches, TripletLoss(), opt, log_wandb=False)
    assert avg == avg and model.training and model.query_tower.pretrained_model.training
    assert torch.equal(model.query_tower.pool_tokens({"input_ids": ids, "attention_mask": mask}), want)


def test_a_trained_encoder_with_dropout_is_refused_in_train_mode():
    from two_towers_overlords_amd.encoder import PackedBertEncoder

    model = two_towers(bert(dropout=0.1), train_encoder=True)
    ids, mask = texts()
    model.encode_query_ids(ids, mask)
    model.train()
    for f in (lambda: model.encode_query_ids(ids, mask), lambda: PackedBertEncoder(bert(dropout=0.1).train())(ids, mask)):
        with pytest.raises(RuntimeError, match="dropout"):
            f()
