"""The selective model's parameters in the training's optimiser (CPU)."""

import torch


class _Config:
    input_size, hidden_layers, output_size, bias = 8, [32, 32], 4, True
    lr_w, lr_positions, weight_decay = 1e-2, 5e-2, 1e-1


def test_rates_and_step_sizes_do_not_decay():
    from delrec.networks import RNN_gated, RNN_selective
    from delrec.training.mem import make_optimizer
    model = RNN_selective(_Config)
    opt = make_optimizer(model, _Config)
    weights, positions, kept = opt.param_groups
    assert weights['weight_decay'] == 1e-1 and positions['params'] == [] and kept['weight_decay'] == 0.0 and kept['lr'] == 1e-2
    free = {id(p) for p in kept['params']}
    for name, p in model.named_parameters():
        assert (id(p) in free) == name.endswith(('A_log', '.D', 'dt_bias')), name
    assert len(weights['params']) + len(kept['params']) == len(list(model.parameters()))
    # a step without gradients' pull: decay alone moves a parameter
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    for p in model.parameters():
        p.grad = torch.zeros_like(p)
    opt.step()
    for name, p in model.named_parameters():
        moved = not torch.equal(p, before[name])
        assert moved == (id(p) not in free and bool(before[name].any())), name
    # models without such parameters keep their two groups
    assert len(make_optimizer(RNN_gated(_Config), _Config).param_groups) == 2
