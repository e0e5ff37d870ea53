"""Rotary positions, frame-causal attention and Muon under data parallelism: 2 ranks x B/2 clips reproduce 1 rank x B, and the split
and the in-library paths walk the one-call step's trajectory.  The ranks share the one GPU and exchange through gloo."""
import os
import socket

import numpy as np
import pytest
import torch.multiprocessing as mp

from tests.util import make_case

pytestmark = pytest.mark.gpu
T = 3
SHAPE, PATCH, D, H, L, B, AXES = (4, 3, 16, 16), 4, 64, 2, 2, 4, [8, 12, 12]
LR = 0.02


def build(images=slice(None)):
    import cora_amd as ca
    case = make_case(SHAPE, PATCH, D, H, L, B, seed=23, clip_h=3.0, clip_w=0.5)
    hp = case["hp"]
    case["x"], case["h"] = case["x"][images], [t[images] for t in case["h"]]
    cfg = ca.TransformerConfig(image_shape=SHAPE, hidden_size=D, num_heads=H, num_blocks=L, patch_size=PATCH, theta=100, axes_dim=AXES,
                               use_noise=True, use_inference_lr_scaling=hp.use_scaling, inference_lr_scale_base=hp.scale_base,
                               use_status_init_in_training=False, update_weights_every_inference_step=False,
                               pos_encoding="rotary", causal_frames=True)
    model = ca.TransformerDecoder(cfg)
    model.set_weights(case["W"])
    for l, t in enumerate(case["h"]):
        model.vodes[l].h.set(t)
    oh = ca.Optim(lambda: ca.chain(ca.clip_by_global_norm(hp.clip_h), ca.sgd(0.095, momentum=hp.momentum)))
    # coefficients that raise no singular value's error by more than 1.5 a step
    muon = ca.muon(LR, ns_steps=2, ns_coeffs=(1.5, -0.5, 0.0))
    return model, case, ca.Optim(lambda: ca.chain(ca.clip_by_global_norm(hp.clip_w), muon), model), oh


def result(model, case, ow, oh, batches=1):
    import cora_amd as ca
    outs = [ca.train_on_batch(T, case["x"], model=model, optim_w=ow, optim_h=oh) for _ in range(batches)]
    return [float(o[0]) for o in outs], [model.vodes[l].h.get() for l in range(L + 2)], model.get_weights()


def same_updates(got, want, before):
    """Vodes agree to 2e-5; gradients, sums over tokens of products of two such, to 1e-4; two steps raise that to 2.3e-4 of a block
    matrix' update.  AdamW's first step, g / |g|, turns the rounding of small gradients into that of the step: as much as that of
    the weights' largest value."""
    for k, w in want.items():
        if np.ndim(w) == 2 and "transformer_blocks" in k:
            assert np.linalg.norm(got[k] - w) <= 2.3e-4 * np.linalg.norm(w - before[k]) + 2.0 ** -23 * np.linalg.norm(w), k
        else:
            assert np.abs(got[k] - w).max() <= 2e-4 * np.abs(w).max() + 1e-6 * LR / 1e-3, k


def _worker(rank, world, port, q):
    import torch.distributed as dist
    from cora_amd.dist import DataParallel, shard_slice
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    model, case, ow, oh = build(shard_slice(B, rank, world))
    DataParallel(model, B // world, exact_clip=True)
    q.put((rank,) + result(model, case, ow, oh))
    dist.barrier()
    model.close()
    dist.destroy_process_group()


def test_two_ranks_match_one_rank():
    model, case, ow, oh = build()
    energies, h, w = result(model, case, ow, oh)
    model.close()
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = sorted([q.get(timeout=60) for _ in procs], key=lambda r: r[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    for l in range(L + 2):
        got = np.concatenate([r[2][l] for r in res])
        assert np.abs(got - h[l]).max() <= 2e-5 * np.abs(h[l]).max(), l
    assert abs(res[0][1][0] + res[1][1][0] - energies[0]) <= 1e-5 * abs(energies[0])
    for k in w:
        assert np.array_equal(res[0][3][k], res[1][3][k]), k
    same_updates(res[0][3], w, case["W"])


@pytest.mark.parametrize("backend", ["torch", "rccl"])
def test_one_rank_walks_the_one_call_step(backend):
    """Several batches, so that eager launches and captured graphs both run."""
    from cora_amd.dist import DataParallel
    runs = []
    for parallel in (False, True):
        model, case, ow, oh = build()
        if parallel:
            DataParallel(model, B, backend=backend, exact_clip=True)
        runs.append(result(model, case, ow, oh, 1) + result(model, case, ow, oh, 3))
        model.close()
    (e1, h1, w1, e4, h4, w4), (f1, g1, v1, f4, g4, v4) = runs
    assert np.allclose(e1 + e4, f1 + f4, rtol=1e-5)
    for a, b in zip(h1 + h4, g1 + g4):
        assert np.abs(a - b).max() <= 1e-4 * np.abs(a).max()
    same_updates(v1, w1, case["W"])
    for k in w4:
        assert np.abs(w4[k] - v4[k]).max() <= 1e-3 * max(np.abs(w4[k]).max(), 1e-2), k
