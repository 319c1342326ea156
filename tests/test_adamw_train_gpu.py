"""optimizer_type = adamw through the models' train_op: the variables against a 64-bit AdamW on the model's own gradients."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _model(seed=3, **over):
    from avsi_amd import models
    B, N = 4, 2880
    T = N // 192
    rng = np.random.default_rng(seed)
    wav = np.clip(np.round(rng.normal(0, 3000, size=(B, N))), -32768, 32767).astype(np.float32)
    masks = np.ones((B, T, 257), dtype=np.float32)
    masks[:, 4:7] = 0
    cfg = dict(audio_feat_dim=257, video_feat_dim=136, audio_len=N, net_dim=[250, 250, 250], optimizer_type='adamw', weight_decay=0.05,
               starter_learning_rate=1e-3, lr_updating_steps=2, lr_decay=0.5, batch_size=B, l2=0.0)
    cfg.update(over)
    mean, std = np.zeros(257, dtype=np.float32), np.ones(257, dtype=np.float32)
    m = models.StackedBLSTMModel(np.full(B, T), wav, masks, mean, std, 0.0, cfg, input='a', seed=5)
    return m, dict(sequence_lengths=np.full(B, T), target_sources=wav, masks=masks)


def test_three_adamw_steps(tmp_path):
    m, feed = _model()
    v = m.variables
    w = v.flat.double().clone()
    mo, ve = torch.zeros_like(w), torch.zeros_like(w)
    decay = torch.zeros_like(w)
    for _, shape, off in m.layout.ref_entries:
        if len(shape) > 1:
            decay[off:off + int(np.prod(shape))] = 0.05
    bound = torch.zeros_like(w)
    rates = []
    for step in (1, 2, 3):
        m.feed(**feed)
        g = m.gradients.double()
        lr = m.learning_rate
        rates.append(lr)
        mo, ve = 0.9 * mo + 0.1 * g, 0.999 * ve + 0.001 * g * g
        d = torch.sqrt(ve / (1 - 0.999 ** step)) + 1e-8
        up = mo / (1 - 0.9 ** step) / d
        # (what a step may add: see test_adamw_gpu; the moments' own roundings add up over the steps, m's relative to its terms)
        bound = bound + lr * (18 * U * step / (1 - 0.9 ** step) * torch.maximum(mo.abs(), 0.1 * g.abs()) / d + 40 * U * up.abs()) + 3 * U * w.abs() + 1e-12
        w = w - lr * (up + decay * w)
        assert m.train_op is None and m.global_step == step
    assert rates == [1e-3, 1e-3, 5e-4]
    # a first moment that cancels over the steps keeps the roundings of its terms: allow those of the largest gradient in its place
    assert bool(((v.flat.double() - w).abs() <= 8 * bound + 2e-9).all())
    assert v._adamw is not None and torch.equal(v.adam_m, torch.cat([t.reshape(-1) for t in v._adamw[1].state['m']]))
    # a checkpoint restores slots and goes on alike
    path = v.save(str(tmp_path / 'ck'))[:-4]
    m2, _ = _model()
    m2.variables.restore(path)
    m2.learning_rate
    for mm in (m, m2):
        mm.feed(**feed)
        mm.train_op
    assert torch.equal(m.variables.flat, m2.variables.flat) and m2.global_step == 4


def test_adamw_refuses_an_l2_term_and_obeys_the_guard():
    m, feed = _model(l2=1e-3)
    m.feed(**feed)
    with pytest.raises(ValueError, match="l2 must be 0"):
        m.train_op
    m, feed = _model()
    m.feed(**feed)
    before = m.variables.flat.clone()
    m.apply_gradients(torch.ones_like(before), guard=torch.tensor([float('nan'), 0.0], device='cuda'))
    assert torch.equal(m.variables.flat, before) and bool((m.variables.adam_m == 0).all())
