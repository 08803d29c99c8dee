"""What load_state_dict of FusedAdamW and FusedClipAdam does to the moments that exist, on the host: a step recorded in a
HIP graph holds their addresses, so no load may free them."""
import pytest
import torch

from recommend_amd.optim import FusedAdamW, FusedClipAdam, encode_moment


def optimizer(bits, shapes=((100, 64), (64,), ())):
    """With moments as a step makes them (steps need a GPU)."""
    g = torch.Generator().manual_seed(1)
    params = [torch.nn.Parameter(torch.randn(s, generator=g)) for s in shapes]
    opt = FusedAdamW(params, state_bits=bits)
    for p in params:
        m, v = torch.randn(p.shape, generator=g), torch.rand(p.shape, generator=g)
        if opt._is8(p):
            st = dict(zip(("exp_avg8", "exp_avg8_scale"), encode_moment(m)))
            st.update(zip(("exp_avg_sq8", "exp_avg_sq8_scale"), encode_moment(v, True)))
        else:
            st = {"exp_avg": m, "exp_avg_sq": v}
        opt.state[p].update(st, step=torch.tensor(3.0))
    return opt, params


def addresses(opt, p):
    return {k: v.data_ptr() for k, v in opt.state[p].items() if k != "step"}


def cleared(opt, p):
    return all(bool((v.float() == 0).all()) for k, v in opt.state[p].items() if k != "step")


@pytest.mark.parametrize("bits", [8, 32])
def test_a_checkpoint_from_before_the_first_step_clears_in_place(bits):
    opt, params = optimizer(bits)
    first = FusedAdamW([torch.nn.Parameter(p.detach().clone()) for p in params], state_bits=bits).state_dict()
    assert not first["state"]
    held = [addresses(opt, p) for p in params]
    opt.load_state_dict(first)
    assert [addresses(opt, p) for p in params] == held and all(held)
    assert all(cleared(opt, p) for p in params) and opt._restored_step == 0


@pytest.mark.parametrize("bits", [8, 32])
def test_a_checkpoint_without_one_parameter_clears_that_one(bits):
    opt, params = optimizer(bits)
    saved = optimizer(bits)[0].state_dict()
    want = {k: v.clone() for k, v in saved["state"][1].items()}
    saved["state"][0] = {"momentum_buffer": torch.ones(100, 64)}          # another optimizer's
    del saved["state"][2]
    held = [addresses(opt, p) for p in params]
    opt.load_state_dict(saved)
    assert [addresses(opt, p) for p in params] == held
    assert cleared(opt, params[0]) and cleared(opt, params[2]) and "momentum_buffer" not in opt.state[params[0]]
    assert all(torch.equal(opt.state[params[1]][k], v) for k, v in want.items())
    assert opt._restored_step == 3


def test_buffers_that_cannot_be_used_again_are_not_freed():
    """Moments of another form than the checkpoint's become (the threshold was moved): a recorded step still has them."""
    opt, params = optimizer(8)
    saved = optimizer(8)[0].state_dict()
    old = {v.data_ptr() for k, v in opt.state[params[0]].items() if k != "step"}
    opt.min_8bit_size = 1 << 20
    opt.load_state_dict(saved)
    assert set(opt.state[params[0]]) == {"step", "exp_avg", "exp_avg_sq"}
    assert old <= {t.data_ptr() for t in opt._held}


def test_a_checkpoint_of_other_sizes_leaves_everything_as_it_was():
    opt, params = optimizer(32)
    held = [addresses(opt, p) for p in params]
    values = [v.clone() for p in params for v in opt.state[p].values()]
    for bits in (8, 32):
        with pytest.raises(ValueError, match="does not fit"):
            opt.load_state_dict(optimizer(bits, ((100, 66), (64,), ()))[0].state_dict())
    with pytest.raises(ValueError):
        opt.load_state_dict(optimizer(32, ((100, 64),))[0].state_dict())
    assert [addresses(opt, p) for p in params] == held
    assert all(torch.equal(a, b) for a, b in zip([v for p in params for v in opt.state[p].values()], values))


def test_counts_that_differ_continue_with_the_largest():
    w = [torch.nn.Parameter(torch.ones(3)) for _ in range(2)]
    theirs = torch.optim.AdamW(w)
    for k in range(4):
        w[0].grad, w[1].grad = torch.ones(3), torch.ones(3) if k == 3 else None
        theirs.step()
    assert [int(theirs.state[p]["step"]) for p in w] == [4, 1]
    opt = FusedAdamW([torch.nn.Parameter(torch.ones(3)) for _ in range(2)])
    opt.load_state_dict(theirs.state_dict())
    assert opt._restored_step == 4


def test_clip_adam_keeps_moments_that_the_checkpoint_lacks():
    params = [torch.nn.Parameter(torch.ones(n)) for n in (5, 6, 7)]
    opt = FusedClipAdam(params)
    for p in params:
        opt.state[p].update(exp_avg=torch.full_like(p, 2.0), exp_avg_sq=torch.full_like(p, 3.0), step=torch.tensor(3.0))
    held = [addresses(opt, p) for p in params]
    partial = opt.state_dict()
    partial["state"] = {1: {k: v.clone() for k, v in partial["state"][1].items()}}
    opt.load_state_dict(partial)
    assert [addresses(opt, p) for p in params] == held
    assert cleared(opt, params[0]) and cleared(opt, params[2]) and bool((opt.state[params[1]]["exp_avg"] == 2).all())
    opt.load_state_dict(FusedClipAdam([torch.nn.Parameter(torch.ones(n)) for n in (5, 6, 7)]).state_dict())
    assert [addresses(opt, p) for p in params] == held and all(cleared(opt, p) for p in params)
    assert opt._restored_step == 0


@pytest.mark.parametrize("other", ["amsgrad", "maximize"])
def test_other_updates_than_the_built_one_are_refused(other):
    """torch's AdamW with them takes other steps: neither its checkpoints nor groups that ask for them pass in silence."""
    w = torch.nn.Parameter(torch.ones(3))
    theirs = torch.optim.AdamW([w], **{other: True})
    w.grad = torch.ones(3)
    theirs.step()
    opt, params = optimizer(32, ((3,),))
    held = addresses(opt, params[0])
    with pytest.raises(ValueError, match=other):
        opt.load_state_dict(theirs.state_dict())
    assert addresses(opt, params[0]) == held and opt.param_groups[0]["lr"] == 1e-3
    with pytest.raises(ValueError, match=other):
        FusedAdamW([{"params": [w], other: True}])
    bad = torch.optim.AdamW([w]).state_dict()
    bad["param_groups"][0]["betas"] = (0.9, 1.0)
    with pytest.raises(ValueError, match="betas"):
        opt.load_state_dict(bad)


def test_a_refused_group_is_not_added():
    opt, _ = optimizer(32, ((3,),))
    with pytest.raises(ValueError, match="betas"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(2))], "betas": (0.9, 1.0)})
    assert len(opt.param_groups) == 1


def test_moments_are_converted_one_parameter_at_a_time(monkeypatch):
    """A checkpoint takes the memory of one parameter's moments beside those that exist, not of all."""
    opt, params = optimizer(32, ((100, 64), (100, 64), (100, 64)))
    saved, alive, most = optimizer(8, ((100, 64), (100, 64), (100, 64)))[0].state_dict(), [], []
    make = FusedAdamW._moments_of

    def watched(self, p, src):
        st = make(self, p, src)
        import weakref
        alive.extend(weakref.ref(t) for k, t in st.items() if k != "step")
        most.append(sum(r() is not None for r in alive))
        return st

    monkeypatch.setattr(FusedAdamW, "_moments_of", watched)
    opt.load_state_dict(saved)
    assert len(most) == 3 and max(most) <= 4         # this parameter's two, and the last one's still in a variable
