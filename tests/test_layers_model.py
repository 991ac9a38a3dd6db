"""BERT on the package's own layers: the same model as on torch's, and trained as a job."""
import pytest
import torch

from hipress_b200 import HipressConfig
from hipress_b200.models import bert_tiny
from hipress_b200.models.bert import BertConfig


def pair(device):
    torch.manual_seed(0)
    plain = bert_tiny(dropout=0.0).to(device)
    fused = bert_tiny(dropout=0.0, fused=True).to(device)
    fused.load_state_dict(plain.state_dict())
    ids = torch.randint(0, 1000, (3, 40), device=device)
    labels = torch.where(torch.rand(3, 40, device=device) < 0.3, ids, -100)
    mask = torch.arange(40, device=device)[None] < torch.tensor([[40], [17], [31]], device=device)
    return plain, fused, ids, torch.where(mask, labels, -100), mask


def grads(model, *a, **kw):
    loss = model(*a, **kw)
    loss.backward()
    return loss.detach(), {n: p.grad for n, p in model.named_parameters() if p.grad is not None}


def test_fused_layers_are_the_model():
    plain, fused, ids, labels, mask = pair("cpu")
    want, wg = grads(plain, ids, labels, key_mask=mask)
    got, gg = grads(fused, ids, labels, key_mask=mask)
    assert torch.allclose(got, want, rtol=1e-5)
    assert wg.keys() == gg.keys()
    for n in wg:   # 32 bits, sums in another order
        assert torch.allclose(gg[n], wg[n], rtol=1e-4, atol=1e-6 + 1e-4 * wg[n].abs().max().item()), n
    assert torch.allclose(fused(ids, key_mask=mask)[mask], plain(ids, key_mask=mask)[mask], atol=1e-4)


def test_fused_layers_refuse_dropout_of_probabilities():
    with pytest.raises(ValueError, match="attn_dropout"):
        BertConfig(fused=True)
    c = BertConfig(fused=True, attn_dropout=0.0)
    assert c.dropout == 0.1


def train(device, dtype, **kw):
    from hipress_b200.train.harness import build_job
    cfg = HipressConfig(algorithm="onebit", topology="ring", comp_threshold=1024)
    job = build_job("bert_base", cfg, batch=4, seq_len=32, dtype=dtype, device=device,
                    model_kwargs=dict(hidden=64, layers=2, heads=4, ffn=128, vocab_size=500, attn_dropout=0.0, **kw))
    x, y = job.to_device(*job.host_batch(0))
    losses = [job.step(x, y).item() for _ in range(12)]
    job.optimizer.close()
    return losses


def test_a_job_trains_on_fused_layers():
    losses = train(torch.device("cpu"), torch.float32, fused=True)
    assert losses[-1] < losses[0]


@pytest.mark.gpu
def test_fused_layers_on_the_gpu():
    plain, fused, ids, labels, mask = pair("cuda")
    want, wg = grads(plain, ids, labels, key_mask=mask)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got, gg = grads(fused, ids, labels, key_mask=mask)
    assert abs(got - want) < 0.02 * abs(want)
    assert wg.keys() == gg.keys()
    for n in wg:   # a dozen roundings to bfloat16 in a row, 2^-8 each
        assert (gg[n] - wg[n]).norm() <= 0.05 * wg[n].norm() + 1e-6, n


@pytest.mark.gpu
def test_a_job_trains_on_fused_layers_on_the_gpu():
    losses = train(torch.device("cuda"), torch.bfloat16, fused=True)
    assert losses[-1] < losses[0]
    assert abs(losses[0] - train(torch.device("cuda"), torch.bfloat16)[0]) < 0.05 * losses[0]


@pytest.mark.parametrize("args,what", [(["--model", "vgg19"], "BERT"), (["--model", "resnet50"], "BERT"), (["--model", "transformer"], "BERT"),
                                       (["--model", "bert-base", "--fp32"], "fp32")])
def test_the_launcher_refuses_fused_layers_that_cannot_be(args, what, monkeypatch, capsys):
    from hipress_b200.train import pytorch_imagenet as T
    monkeypatch.setattr(T.torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(T, "build_job", lambda *a, **kw: pytest.fail("a job was built"))
    with pytest.raises(SystemExit) as stop:
        T.main([*args, "--fused-layers"])
    assert stop.value.code == 2
    assert what in capsys.readouterr().err
