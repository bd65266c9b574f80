"""GPU tests of the gated delta rule on values of any size that f32 holds: tiny states under large inputs, inputs that grow or vanish by many powers of two from
one chunk of 64 rows to the next, columns that a decay has cleared. Against the definition in 64 bits (gdn_util.py)."""
import numpy as np
import pytest
import torch

from tests.attn_util import check, f64
from tests.gdn_util import D, Rows, rule
from tests.gpu_util import say
from tests.test_gpu_gdn import workspace

pytestmark = pytest.mark.gpu


def sized(r, sizes, state=None):
    """Value rows of sizes[i] for the i-th 64 rows of every sequence; states of a size."""
    t = r.front
    for n in r.lens:
        for i in range(n):
            r.rows[t + i, 2 * r.kh * D:(2 * r.kh + r.heads) * D] *= sizes[min(i // 64, len(sizes) - 1)]
        t += n
    if state is not None:
        r.state = r.state * state if state else torch.zeros_like(r.state)
    return r


def parts(r, t, n):
    x, ab, keys = f64(r.rows[t:t + n].float()), f64(r.ab[t:t + n].float()), r.kh * D
    return [x[:, :keys].reshape(n, r.kh, D), x[:, keys:2 * keys].reshape(n, r.kh, D), x[:, 2 * keys:2 * keys + r.heads * D].reshape(n, r.heads, D), ab[:, :r.heads],
            ab[:, r.heads:2 * r.heads], f64(r.a_log), f64(r.dt_bias)]


def compare(r, was, chunked, size):
    """Every sequence against the rule. Answers and states are linear in the states and value rows: the rule is taken of these over `size`, so that the least
    tolerance of its own is one of that size."""
    t = r.front
    for s, n in enumerate(r.lens):
        p, x = int(r.slot[s]), parts(r, t, n)
        x[2] = x[2] / size
        want, tol, states, tols = rule(*x, was[p] / size, r.eps, r.scale, chunked)
        check(f64(r.out[t:t + n].float()) / size, want, tol, f"rows of sequence {s}")
        check(f64(r.state[p]) / size, states[-1], np.broadcast_to(tols[-1], states[-1].shape), f"state of sequence {s}")
        t += n


@pytest.mark.parametrize("chunked", [False, True])
@pytest.mark.parametrize("state,sizes", [(1e-36, [300.0]), (1e-40, [300.0]), (2.0 ** -96, [2.0 ** 25]), (2.0 ** -120, [2.0 ** 100]), (2.0 ** 100, [2.0 ** -100]),
                                         (0, [2.0 ** -120, 300.0]), (0, [2.0 ** -123, 2.0 ** 9, 2.0 ** -60]), (1e-37, [0.0, 2.0 ** 20]), (2.0 ** 60, [2.0 ** 60, 1.0, 2.0 ** 90]),
                                         (2.0 ** -100, [2.0 ** -100])])
def test_values_of_any_size(ctx, state, sizes, chunked):
    say(f"delta rule, states of {state}, values of {sizes}, chunked {chunked}")
    r = sized(Rows(2, 4, [200, 64, 33], seed=50), sizes, state)
    was = f64(r.state)
    r.call(ctx, workspace=workspace(r) if chunked else None)
    torch.cuda.synchronize()
    compare(r, was, chunked, max([state] + sizes))


@pytest.mark.parametrize("chunked", [False, True])
@pytest.mark.parametrize("before,behind", [(2.0 ** 60, 2.0 ** -100), (2.0 ** -110, 2.0 ** 20), (1.0, 2.0 ** -60), (2.0 ** 100, 1.0), (1e-36, 300.0), (1.0, 1.0)])
def test_columns_that_a_decay_has_cleared(ctx, before, behind, chunked):
    """The last row of a chunk clears the state and adds nothing: what follows is as on zeros, whatever size stood there."""
    say(f"delta rule, states of {before} cleared, then values of {behind}, chunked {chunked}")
    r = sized(Rows(1, 3, [64 + 100], seed=51), [before, behind], before)
    r.rows[63, 2 * D:5 * D] = 0
    r.ab[63, :r.heads] = 20000.0
    r.call(ctx, workspace=workspace(r) if chunked else None)
    torch.cuda.synchronize()
    x = parts(r, 64, 100)
    x[2] = x[2] / behind
    want, tol, states, tols = rule(*x, np.zeros((r.heads, D, D)), r.eps, r.scale, chunked)
    check(f64(r.out[64:].float()) / behind, want, tol, "rows behind")
    check(f64(r.state[int(r.slot[0])]) / behind, states[-1], np.broadcast_to(tols[-1], states[-1].shape), "state")


@pytest.mark.parametrize("chunked", [False, True])
def test_values_whose_sizes_have_nothing_in_common(ctx, chunked):
    """Every row, column and state by a power of two of its own."""
    say(f"delta rule, sizes at random, chunked {chunked}")
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        r = Rows(2, 4, [300, 70], seed=52 + seed, a_at=(0.0, -4.0, 3.0)[seed])
        rows, columns = torch.randint(-40, 41, (r.tokens, 1), generator=g), torch.randint(-40, 41, (1, r.heads * D), generator=g)
        v = slice(2 * r.kh * D, (2 * r.kh + r.heads) * D)
        r.rows[:, v] = (r.rows[:, v].float() * torch.exp2((rows + columns).float()).cuda()).bfloat16()
        r.state *= torch.exp2(torch.randint(-40, 41, (r.slots, r.heads, 1, D), generator=g).float()).cuda()
        was = f64(r.state)
        r.call(ctx, workspace=workspace(r) if chunked else None)
        torch.cuda.synchronize()
        compare(r, was, chunked, 1.0)


@pytest.mark.parametrize("chunked", [False, True])
@pytest.mark.parametrize("state,sizes", [(1.0, [2.0 ** 118]), (0, [2.0 ** 112, 1.0]), (2.0 ** 118, [1.0, 2.0 ** 118])])
def test_values_near_the_end_of_f32(ctx, state, sizes, chunked):
    """Decays of a while together, of which a row's update may not be taken back out of f32's range."""
    say(f"delta rule, states of {state}, values of {sizes}, chunked {chunked}")
    r = sized(Rows(2, 4, [100, 30], a_at=-3.0, seed=56), sizes, state)
    was = f64(r.state)
    r.call(ctx, workspace=workspace(r) if chunked else None)
    torch.cuda.synchronize()
    compare(r, was, chunked, max([state] + sizes))


@pytest.mark.parametrize("chunked", [False, True])
def test_gates_whose_factors_pass_f32(ctx, chunked):
    """exp(a_log) that is no f32 times a softplus that is none, whose product is a decay like any other; sums of a and dt_bias past f32."""
    say(f"delta rule, gates at the ends of f32, chunked {chunked}")
    r = Rows(1, 6, [90, 20], seed=57)
    r.a_log.copy_(torch.tensor([100.0, 95.0, -200.0, 90.0, -104.0, 30.0]))
    r.dt_bias.copy_(torch.tensor([-105.0, 0.0, 3e38, -3e38, 3e38, -31.0]))
    r.ab[:, 2], r.ab[:, 3] = 3e38, -3e38
    for h, most in ((0, 2), (4, 0), (5, 3)):
        r.ab[:, h] = torch.arange(r.tokens, device="cuda").remainder(most + 1).bfloat16()
    was = f64(r.state)
    r.call(ctx, workspace=workspace(r) if chunked else None)
    torch.cuda.synchronize()
    compare(r, was, chunked, 1.0)


@pytest.mark.parametrize("chunked", [False, True])
@pytest.mark.parametrize("before,behind", [(2.0 ** 60, 2.0 ** -100), (2.0 ** 20, 2.0 ** -120), (2.0 ** -110, 2.0 ** 90)])
def test_columns_that_stay_empty_for_a_while(ctx, before, behind, chunked):
    """Cleared, then a whole chunk without inputs, in some columns two, then values of another size; columns that never hold anything stay exactly that."""
    say(f"delta rule, states of {before} cleared and left empty, then values of {behind}, chunked {chunked}")
    r = sized(Rows(1, 3, [64 * 4 + 20], seed=58), [before, 0.0, behind], before)
    v = r.rows[:, 2 * D:5 * D].view(-1, 3, D)
    v[63] = 0
    v[:192, :, 5::16] = 0
    v[:, :, 7::32] = 0
    r.state[:, :, :, 7::32] = 0
    r.ab[63, :r.heads] = 20000.0
    r.call(ctx, workspace=workspace(r) if chunked else None)
    torch.cuda.synchronize()
    x = parts(r, 64, 4 * 64 + 20 - 64)
    x[2] = x[2] / behind
    want, tol, states, tols = rule(*x, np.zeros((r.heads, D, D)), r.eps, r.scale, chunked)
    # (bf16's steps below 2^-126 are 2^-133: an answer is rounded by as much as half of that, of values of 2^-120 that is 2^-14)
    check(f64(r.out[64:].float()) / behind, want, tol + 2.0 ** -134 / behind, "rows behind")
    check(f64(r.state[int(r.slot[0])]) / behind, states[-1], np.broadcast_to(tols[-1], states[-1].shape), "state")
    assert (r.out[:, :, 7::32] == 0).all() and (r.state[int(r.slot[0]), :, :, 7::32] == 0).all()
