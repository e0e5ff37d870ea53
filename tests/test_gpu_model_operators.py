"""The model's own use of the stand-alone operators: rotary positions and frame-causal attention inside the PC step, against
the 64-bit oracle with its attention replaced by the same definition; the Muon weight step against the formula in 64 bits."""
import math

import numpy as np
import pytest
import torch

from oracle import pcvit_ref as R
from tests.operator_bounds import ortho_bound, ortho_ref
from tests.util import make_case, relerr

# (image shape, patch, D, H, L, B, axes or None, causal frames, vode LayerNorms)
CASES = {
    "images_rotary": ((3, 16, 24), 4, 64, 2, 2, 3, [16, 16], False, False),
    "images_rotary_64_tokens": ((3, 32, 32), 4, 64, 1, 2, 2, [24, 32], False, False),     # the fused kernels' shape
    "clips_rotary": ((3, 3, 16, 16), 4, 48, 2, 1, 2, [8, 8, 8], False, False),
    "clips_causal": ((4, 3, 16, 16), 4, 64, 1, 2, 2, None, True, False),                  # the row-tile kernels' shape
    "clips_rotary_causal": ((5, 3, 12, 16), 4, 64, 2, 2, 3, [4, 16, 10], True, False),
    "clips_rotary_causal_vln": ((4, 3, 8, 8), 4, 96, 3, 2, 2, [16, 8, 8], True, True),
}


def oracle_mha(dims, axes, causal, theta):
    """The oracle's attention with queries and keys turned and the future frames hidden."""
    def turn(t):
        if axes is None:
            return t
        shape = dims.image_shape
        frames, hp, wp = (shape[0] if len(shape) == 4 else 1), shape[-2] // dims.patch_size, shape[-1] // dims.patch_size
        grid = torch.meshgrid(torch.arange(frames), torch.arange(hp), torch.arange(wp), indexing="ij")
        pos = [g.reshape(-1).double() for g in grid][3 - len(axes):]
        cols, start = [], 0
        for p, n in zip(pos, axes):
            for i in range(n // 2):
                a = p * theta ** (-2.0 * i / n)
                u, v = t[..., start + 2 * i], t[..., start + 2 * i + 1]
                cols += [u * a.cos() - v * a.sin(), u * a.sin() + v * a.cos()]
            start += n
        return torch.cat([torch.stack(cols, -1), t[..., start:]], -1)

    def mha(xn, Wq, Wk, Wv, Wo, H):
        Bn, N, D = xn.shape
        q, k, v = [R.linear(xn, w).reshape(Bn, N, H, D // H).transpose(1, 2) for w in (Wq, Wk, Wv)]
        s = turn(q) @ turn(k).transpose(-1, -2) / math.sqrt(D // H)
        if causal:
            frame = torch.arange(N) // (N // dims.image_shape[0])
            s = s.masked_fill(frame[None, :] > frame[:, None], -math.inf)
        return R.linear((torch.softmax(s, -1) @ v).transpose(1, 2).reshape(Bn, N, D), Wo)
    return mha


def setup(name, monkeypatch, optim_w=None, compute_dtype="fp32", ipc=False):
    import cora_amd as ca
    shape, patch, D, H, L, B, axes, causal, vln = CASES[name]
    case = make_case(shape, patch, D, H, L, B, seed=11, vode_ln=vln)
    d, hp = case["dims"], case["hp"]
    if axes:
        case["pos"] = np.zeros_like(case["pos"])
    monkeypatch.setattr(R, "mha", oracle_mha(d, axes, causal, 100.0))
    cfg = ca.TransformerConfig(
        image_shape=shape, hidden_size=D, num_heads=H, num_blocks=L, patch_size=patch, theta=100, axes_dim=axes or [2, 2, 2],
        use_noise=True, use_inference_lr_scaling=hp.use_scaling, inference_lr_scale_base=hp.scale_base,
        update_weights_every_inference_step=ipc, use_status_init_in_training=False, use_vode_state_layernorm=vln,
        pos_encoding="rotary" if axes else "sinusoidal", causal_frames=causal)
    model = ca.TransformerDecoder(cfg, compute_dtype=compute_dtype)
    if axes:
        assert not model.positional_embedding.any()
    else:
        model.positional_embedding = case["pos"]
    model.set_weights(case["W"])
    for l, t in enumerate(case["h"]):
        model.vodes[l].h.set(t)
    oh = ca.Optim(lambda: ca.chain(ca.clip_by_global_norm(hp.clip_h), ca.sgd(0.095, momentum=hp.momentum)))
    base = optim_w or ca.adamw(1e-3, weight_decay=hp.wd)
    ow = ca.Optim(lambda: ca.chain(ca.clip_by_global_norm(hp.clip_w), base), model)
    return ca, case, model, ow, oh


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CASES))
def test_train_on_batch_matches_the_oracle(name, monkeypatch):
    """Three batches: eager launches, then graph replays; vodes, energies, gradients, weights and the reconstruction."""
    ca, case, model, ow, oh = setup(name, monkeypatch)
    T, W, h, adam = 3, case["W"], case["h"], R.AdamState()
    for batch in range(3):
        ref = R.train_on_batch(T, case["x"], W, h, case["pos"], case["dims"], case["hp"], [0.095] * T, 1e-3, adam=adam)
        Eh, Ew, gh, gw, mse = ca.train_on_batch(T, case["x"], model=model, optim_w=ow, optim_h=oh)
        assert model.kernel_path() == "per-op"
        assert relerr(ca.step_energies(model, T)[0], ref["energies"]) < 1e-4
        for l in range(case["dims"].L + 2):
            assert relerr(model.vodes[l].h.get(), ref["h"][l]) < 1e-4, l
            assert relerr(gh[l], ref["final_h_grad"][l]) < 1e-3, l
        for k, g in ref["w_grad"].items():
            assert relerr(gw[k], g) < 1e-3, k
        assert abs(mse - ref["train_mse"]) <= 1e-4 * ref["train_mse"]
        W, h = ref["weights"], [t for t in ref["h"]]
        model.set_weights({k: v.astype(np.float32) for k, v in W.items()})    # AdamW's first steps amplify rounding
        for l, t in enumerate(h):
            model.vodes[l].h.set(t.astype(np.float32))
    with ca.step(model, ca.STATUS.INIT):
        ca.forward(case["x"], model=model)
    with ca.step(model, ca.STATUS_FORWARD):
        xhat = ca.forward(None, model=model)
    h0 = model.vodes[0].h.get()
    want = R.init_vodes(h0, W, case["pos"], case["dims"])
    for l in range(1, case["dims"].L + 2):
        assert relerr(model.vodes[l].h.get(), want[l]) < 1e-4, l
    assert np.isfinite(xhat).all()
    model.close()


@pytest.mark.gpu
@pytest.mark.parametrize("name,mode,bar", [("clips_rotary_causal", "bf16", 1e-2), ("images_rotary", "bf16", 1e-2), ("clips_rotary_causal", "bf16x3", 1e-4)])
def test_other_compute_dtypes(name, mode, bar, monkeypatch):
    ca, case, model, ow, oh = setup(name, monkeypatch, compute_dtype=mode)
    ref = R.train_on_batch(3, case["x"], case["W"], case["h"], case["pos"], case["dims"], case["hp"], [0.095] * 3, 1e-3)
    ca.train_on_batch(3, case["x"], model=model, optim_w=ow, optim_h=oh)
    assert relerr(ca.step_energies(model, 3)[0], ref["energies"]) < bar
    for l in range(case["dims"].L + 2):
        assert relerr(model.vodes[l].h.get(), ref["h"][l]) < bar, l
    model.close()


BLOCK = ("query_proj.weight", "key_proj.weight", "value_proj.weight", "output_proj.weight", "linear1.nn.weight", "linear2.nn.weight")


def muon_step(W, grads, mom, recipe, lr, gscale):
    """W and mom after one step of every block matrix, in 64 bits from the given gradients."""
    new, tol = {}, {}
    for k, g in grads.items():
        if not k.endswith(BLOCK):
            continue
        g = torch.from_numpy(g).double() * gscale
        mom[k] = recipe.beta * mom.get(k, torch.zeros_like(g)) + g
        u = g + recipe.beta * mom[k] if recipe.nesterov else mom[k]
        coef = recipe.coefficients()
        O = ortho_ref(u, recipe.ns_steps, coef, recipe.eps)
        size = math.sqrt(max(1.0, g.shape[0] / g.shape[1]))
        w = torch.from_numpy(W[k]).double()
        new[k] = w - lr * (size * O + recipe.weight_decay * w)
        # u is rounded to fp32 (2^-23 with its sum): of that size again what the iteration makes of it
        tol[k] = lr * size * 2 * ortho_bound(u, recipe.ns_steps, coef, recipe.eps, torch.float32) * O.norm() + 2.0 ** -23 * w.norm()
    return new, tol


@pytest.mark.gpu
@pytest.mark.parametrize("name,kw", [
    ("clips_rotary_causal", dict(weight_decay=0.01)), ("images_rotary_64_tokens", dict(nesterov=False)),
    ("clips_causal", dict(ns_steps=3, ns_coeffs=((3.4445, -4.775, 2.0315), (2.5, -2.25, 0.75), (1.875, -1.25, 0.375)), beta=0.5))])
def test_muon_weight_step(name, kw, monkeypatch):
    """All three operators in the model's training step; momentum over three batches, the last ones as graph replays."""
    import cora_amd as ca
    recipe = ca.muon(0.02, **kw)
    ca, case, model, ow, oh = setup(name, monkeypatch, optim_w=recipe)
    B, mom, ref_mom = case["x"].shape[0], {}, {}
    adam = R.AdamState()
    for batch in range(3):
        before, h = model.get_weights(), [model.vodes[l].h.get() for l in range(case["dims"].L + 2)]
        ref = R.train_on_batch(2, case["x"], before, h, case["pos"], case["dims"], case["hp"], [0.095] * 2, 0.02)
        _, _, _, gw, _ = ca.train_on_batch(2, case["x"], model=model, optim_w=ow, optim_h=oh)
        grads = {k: gw[k] for k in gw.keys()}
        for k, g in ref["w_grad"].items():
            assert relerr(grads[k], g) < 1e-3, k
        norm = math.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in grads.values())) / B
        gscale = (min(1.0, case["hp"].clip_w / norm)) / B
        want, tol = muon_step(before, grads, mom, recipe, 0.02, gscale)
        after = model.get_weights()
        assert len(want) == 6 * case["dims"].L
        for k, w in want.items():
            assert float((torch.from_numpy(after[k]).double() - w).norm()) <= tol[k], (batch, k)
        # everything else by AdamW, m and v from the same gradients
        adam.count += 1
        for k, g in grads.items():
            if k in want:
                continue
            g = g.astype(np.float64) * gscale
            adam.mu[k] = 0.9 * adam.mu.get(k, 0.0) + 0.1 * g
            adam.nu[k] = 0.999 * adam.nu.get(k, 0.0) + 0.001 * g * g
            upd = adam.mu[k] / (1 - 0.9 ** adam.count) / (np.sqrt(adam.nu[k] / (1 - 0.999 ** adam.count)) + 1e-8)
            assert relerr(after[k], before[k] - 0.02 * upd) < 1e-5, (batch, k)
    # back to AdamW for all: the next step moves the matrices by at most lr (1 + wd |w|)
    ow2 = ca.Optim(lambda: ca.chain(ca.adamw(1e-3, weight_decay=0.0)), model)
    before = model.get_weights()
    ca.train_on_batch(2, case["x"], model=model, optim_w=ow2, optim_h=oh)
    after = model.get_weights()
    for k in before:
        assert np.abs(after[k] - before[k]).max() <= 1.01e-3, k
    model.close()


@pytest.mark.gpu
def test_muon_in_ipc_mode_and_through_make_optimizers(monkeypatch):
    import cora_amd as ca
    recipe = ca.muon(0.01)
    ca, case, model, ow, oh = setup("images_rotary", monkeypatch, optim_w=recipe, ipc=True)
    before = model.get_weights()
    _, _, _, gw, mse = ca.train_on_batch(3, case["x"], model=model, optim_w=ow, optim_h=oh)
    after = model.get_weights()
    for k in before:
        if k.endswith(BLOCK):          # three orthogonal steps: at most lr * 1.3 * sqrt(rank) each
            step = np.linalg.norm(after[k] - before[k]) / (0.01 * math.sqrt(max(1, before[k].shape[0] / before[k].shape[1])) * math.sqrt(min(before[k].shape)))
            assert 0.5 < step < 3 * 1.3, (k, step)
    assert np.isfinite(mse)
    model.close()
    cfg = ca.MODEL_CONFIGS["6block"]
    import dataclasses
    ow, _ = ca.make_optimizers(dataclasses.replace(cfg, use_muon_for_weight_optimizer=True))
    assert isinstance(ow._recipe().base, ca.muon) and ow._recipe().base.adam_weight_decay == cfg.weight_decay


@pytest.mark.gpu
def test_set_muon_refuses():
    import cora_amd as ca
    case = make_case((3, 16, 16), 4, 32, 2, 1, 2)
    cfg = ca.TransformerConfig(image_shape=(3, 16, 16), hidden_size=32, num_heads=2, num_blocks=1, patch_size=4)
    model = ca.TransformerDecoder(cfg)
    model.init_vodes(2)
    oh = ca.Optim(lambda: ca.sgd(0.1, momentum=0.1))
    for kw, word in ((dict(beta=1.0), "beta"), (dict(ns_steps=40), "steps"), (dict(ns_coeffs=(9.0, 0.0, 0.0)), "out of range"),
                     (dict(weight_decay=float("nan")), "finite")):
        with pytest.raises(ca._lib.CoraError, match=word):
            ca.train_on_batch(1, case["x"], model=model, optim_w=ca.Optim(lambda: ca.muon(0.1, **kw)), optim_h=oh)
    model.close()


def test_config_refuses_what_the_model_cannot_do():
    import cora_amd as ca
    ok = dict(image_shape=(3, 16, 16), hidden_size=64, num_heads=2, num_blocks=1, patch_size=4)
    clip = dict(ok, image_shape=(2, 3, 16, 16))
    for kw in (dict(ok, pos_encoding="learned"), dict(ok, pos_encoding="rotary", axes_dim=[20, 16]), dict(ok, pos_encoding="rotary", axes_dim=[3, 16]),
               dict(ok, pos_encoding="rotary", axes_dim=[16]), dict(clip, pos_encoding="rotary", axes_dim=[16, 16]), dict(ok, causal_frames=True)):
        with pytest.raises(ValueError):
            ca.TransformerConfig(**kw)
    c = ca.TransformerConfig(**dict(clip, pos_encoding="rotary", axes_dim=[8, 8, 8], causal_frames=True))
    assert c.causal_frames and ca.create_config(hidden_size=64, num_heads=2, pos_encoding="rotary").pos_encoding == "rotary"
    with pytest.raises(ValueError):
        ca.muon(0.1, ns_steps=2, ns_coeffs=((1.0, 0.0, 0.0),)).coefficients()
    with pytest.raises(ValueError):
        ca.chain(ca.muon(0.1), ca.adamw(0.1))


def test_create_attn_refuses():
    import ctypes as C
    from cora_amd import _lib
    lib = _lib.load()
    cfg = _lib.CoraConfig(N=32, P=48, D=32, H=1, M=64, L=1, B=2, C=3, patch=4, Himg=16, Wimg=16, F=2, max_T=4)
    ctx = C.c_void_p()
    axes = lambda *a: (C.c_int32 * 4)(*a)
    for opt, word in ((dict(causal_block=-1), b"causal_block"), (dict(n_axes=1, axes_dim=axes(8)), b"n_axes"), (dict(n_axes=4), b"n_axes"),
                      (dict(n_axes=2, axes_dim=axes(8, 8), theta=100.0), b"clips"), (dict(n_axes=3, axes_dim=axes(8, 8, 8), theta=0.0), b"theta"),
                      (dict(n_axes=3, axes_dim=axes(8, 8, 7), theta=100.0), b"even"), (dict(n_axes=3, axes_dim=axes(16, 8, 16), theta=100.0), b"channels")):
        assert lib.cora_create_attn(C.byref(cfg), C.byref(_lib.CoraAttnOptions(**opt)), 0, C.byref(ctx)) != 0
        assert word in lib.cora_last_error(None), lib.cora_last_error(None)
