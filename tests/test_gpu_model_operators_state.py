"""The state of the model's weight optimisers: recipes taken in turns, models closed and used again."""
import numpy as np
import pytest

from tests.test_gpu_model_operators import setup

pytestmark = pytest.mark.gpu


def step_of(ca, model, case, ow, oh):
    before = model.get_weights()
    ca.train_on_batch(2, case["x"], model=model, optim_w=ow, optim_h=oh)
    after = model.get_weights()
    return {k: after[k] - before[k] for k in before}


def like_a_new_one(name, monkeypatch, recipe, model, case):
    """the step a new model with this one's weights and vodes takes by a recipe"""
    ca, case, other, _, oh = setup(name, monkeypatch, optim_w=recipe)
    other.set_weights(model.get_weights())
    for l in range(case["dims"].L + 2):
        other.vodes[l].h.set(model.vodes[l].h.get())
    d = step_of(ca, other, case, ca.Optim(lambda: ca.chain(recipe), other), oh)
    other.close()
    return d


def test_recipes_taken_in_turns_start_afresh(monkeypatch):
    """Both recipes are built before the first step, so nothing but the change of recipe starts the state anew: the steps after it
    are a new model's, and AdamW's first one moves no weight by more than lr."""
    import cora_amd as ca
    recipes = ca.muon(0.02), ca.adamw(1e-3, weight_decay=0.0)
    ca, case, model, _, oh = setup("clips_rotary_causal", monkeypatch, optim_w=recipes[0])
    muon, adamw = [ca.Optim(lambda r=r: ca.chain(r), model) for r in recipes]
    for turn in range(2):
        for recipe, optim in zip(recipes, (muon, adamw)):
            want = like_a_new_one("clips_rotary_causal", monkeypatch, recipe, model, case)
            got = step_of(ca, model, case, optim, oh)
            for k in want:
                assert np.array_equal(got[k], want[k]), (turn, k)
                assert optim is muon or np.abs(got[k]).max() <= 1.01e-3, (turn, k)
            step_of(ca, model, case, optim, oh)
            assert model.get_adam_state()[2] == 2
    model.close()


def test_a_state_that_was_set_is_kept_by_the_recipe_that_steps_next(monkeypatch):
    """A saved state of Muon, set before the first step of a new model, is used and not cleared."""
    import ctypes as C

    import cora_amd as ca
    from cora_amd import _lib
    recipe = ca.muon(0.02)
    ca, case, model, muon, oh = setup("images_rotary", monkeypatch, optim_w=recipe)
    for _ in range(3):
        step_of(ca, model, case, muon, oh)
    mu, nu, count = model.get_adam_state()
    weights, vodes = model.get_weights(), [model.vodes[l].h.get() for l in range(case["dims"].L + 2)]
    want = step_of(ca, model, case, muon, oh)
    model.close()
    ca, case, model, muon, oh = setup("images_rotary", monkeypatch, optim_w=recipe)
    model.set_weights(weights)
    for l, t in enumerate(vodes):
        model.vodes[l].h.set(t)
    fp = lambda a: a.ctypes.data_as(C.POINTER(C.c_float))
    _lib.check(_lib.load().cora_set_adam_state(model._ctx, fp(mu), fp(nu), count), model._ctx)
    got = step_of(ca, model, case, muon, oh)
    for k in want:
        assert np.array_equal(want[k], got[k]), k
    model.close()


@pytest.mark.parametrize("name", ["images_rotary", "clips_causal"])
def test_a_closed_model_steps_by_its_recipe_again(name, monkeypatch):
    """close() drops the device state; the next batch sets the recipe up again -- Muon's numbers, the clips, AdamW's numbers -- and
    steps as a new model does."""
    import cora_amd as ca
    for recipe in (ca.muon(0.02), ca.adamw(1e-3, weight_decay=0.5)):
        ca, case, model, optim, oh = setup(name, monkeypatch, optim_w=recipe)
        weights = model.get_weights()
        want = step_of(ca, model, case, optim, oh)
        model.close()
        model.set_weights(weights)
        for l, t in enumerate(case["h"]):
            model.vodes[l].h.set(t)
        got = step_of(ca, model, case, optim, oh)
        for k in want:
            assert np.array_equal(want[k], got[k]), k
        model.close()
