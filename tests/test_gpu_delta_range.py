"""How far apart the magnitudes in one sequence may be: the chunked rule keeps the values that it corrects, and the
state's parts, to 2^-28 of M, the largest |v| or |state| of their chunk; the recurrence keeps 32 bits of each.

Tolerance.  Operands of a path from a value to an output (X, U, the state's parts) are off by 2^-28 M / sqrt(3) rms each,
T takes some two of them on, an output the tokens of a chunk with weights |q . k| of a tenth, 64 at most: under
2^-24.5 M scale rms, five of those the largest of some 10^5: 2^-22 M scale beside the rounding of the output.  The
state's entries, sums over the same tokens with weights |k| of a tenth: 2^-22 M too."""
import pytest

from test_gpu_mixers import H, _cu, _delta_case, _delta_ref, _torch

pytestmark = pytest.mark.gpu


def _run(mcv, cuda, inputs, lens):
    scale = inputs[0].shape[-1] ** -0.5
    out, final = mcv.gated_delta_rule(*(x.to(cuda) for x in inputs), cu_seqlens=_cu(lens, cuda), scale=scale, normalize=True)
    want, size, S = _delta_ref(*inputs, lens, scale, True)
    out = out.cpu().double()
    past = want.abs() > 65519                                    # fp16's largest and half a step: infinite, as it has to be
    assert (out[past].isinf()).all()
    return scale, (out - want).abs().masked_fill(past, 0), H * want.abs() + 2.0 ** -24, (final.cpu().double() - S).abs(), want, S


@pytest.mark.parametrize("n", [64, 150, 400])
@pytest.mark.parametrize("M", [1e3, 1e5, 1e7])
def test_large_state_that_decays(mcv, cuda, n, M):
    q, k, v, g, beta, state = _delta_case(n, [n], 2, 2, 128, 64)
    state = state / state.abs().max() * M
    g[1:6] = -8.0
    scale, err, room, off, want, S = _run(mcv, cuda, (q, k, v, g, beta, state), [n])
    assert (err <= room + 2.0 ** -22 * M * scale + 3 * H * want.abs()).all(), (err - room).max() / (M * scale)
    assert (off <= 2.0 ** -22 * M + 2.0 ** -18 * S.abs()).all(), off.max() / M


@pytest.mark.parametrize("n", [64, 150, 400])
@pytest.mark.parametrize("M", [1e3, 6e4])
@pytest.mark.parametrize("at", [0, 40])
def test_one_large_value(mcv, cuda, n, M, at):
    q, k, v, g, beta, state = _delta_case(n, [n], 2, 2, 128, 64)
    v[at, :, 5] = M
    g[at + 1:at + 5] = -8.0
    scale, err, room, off, want, S = _run(mcv, cuda, (q, k, v, g, beta, state), [n])
    assert (err <= room + 2.0 ** -22 * M * scale + 3 * H * want.abs()).all(), (err - room).max() / (M * scale)
    assert (off <= 2.0 ** -22 * M + 2.0 ** -18 * S.abs()).all(), off.max() / M


@pytest.mark.parametrize("M", [1e3, 1e5, 1e7])
def test_the_recurrence_keeps_32_bits(mcv, cuda, M):
    q, k, v, g, beta, state = _delta_case(9, [9], 2, 2, 128, 64)
    state = state / state.abs().max() * M
    g[1:6] = -8.0
    scale, err, room, off, want, S = _run(mcv, cuda, (q, k, v, g, beta, state), [9])
    assert (err[7:] <= room[7:] + 2.0 ** -18 * want[7:].abs().max()).all()
    assert (off <= 2.0 ** -18 * S.abs().max()).all()


@pytest.mark.parametrize("M", [1e3, 1e5, 1e7])
@pytest.mark.parametrize("n", [150, 400])
def test_a_forgotten_state_costs_nothing(mcv, cuda, n, M):
    """Large, and gone in the first tokens; gone in the second chunk too what the first, which holds its values to 2^-28 of
    that state, has left: all later chunks are as if it had not been."""
    q, k, v, g, beta, state = _delta_case(n, [n], 2, 2, 128, 64)
    state = state / state.abs().max() * M
    g[1:6] = g[70:74] = -8.0
    scale, err, room, off, want, S = _run(mcv, cuda, (q, k, v, g, beta, state), [n])
    # one rounding of the outputs, 0.42 H rms, and the two-part operands; the state as everywhere
    assert err[128:].norm() <= 0.6 * H * want[128:].norm() and off.norm() <= 16 * 2.0 ** -22 * S.norm()


@pytest.mark.parametrize("at", [192, 200, 399])
def test_what_comes_later_changes_no_bit(mcv, cuda, at):
    """Outputs of earlier chunks do not depend on later tokens, large ones, infinite ones or none at all."""
    torch = _torch()
    q, k, v, g, beta, state = _delta_case(5, [400], 2, 4, 128, 64)
    run = lambda x, n: mcv.gated_delta_rule(*(t[:n].to(cuda) for t in (q, k, x, g, beta)), state.to(cuda), normalize=True)[0][:192]    # noqa: E731
    want = run(v, 400)
    for value in (60000.0, float("inf"), 0.0):
        x = v.clone()
        x[at:] = value
        assert torch.equal(run(x, 400).view(torch.int16), want.view(torch.int16)), value
    assert torch.equal(run(v, 192).view(torch.int16), want.view(torch.int16))


def test_tiny_and_zero(mcv, cuda):
    """No values for a long while, a state that decays to next to nothing, and values again; all zero."""
    torch = _torch()
    q, k, v, g, beta, state = _delta_case(6, [600], 2, 2, 64, 32)
    v[70:500] = 0
    g[80:500] *= 4
    v[100:] *= 2.0 ** -10
    for inputs in ((q, k, v, g, beta, state), (q, k, v, g, beta, 0 * state)):
        scale, err, room, off, want, S = _run(mcv, cuda, inputs, [600])
        assert (err <= room + 2.0 ** -18 * want.abs()).all() and off.norm() <= 16 * 2.0 ** -22 * S.norm()
    # no value at all: a chunk's M is what decay has left of the state before it, the state's last bits down to 2^-140
    scale, err, room, off, want, S = _run(mcv, cuda, (q, k, 0 * v, g, beta, state * 2.0 ** -30), [600])
    G = torch.cat((0 * g[:1], g)).double().cumsum(0)
    ends = list(range(0, 600, 64)) + [600]
    for h in range(2):
        M = max(float((G[a, h] - G[b, h] + G[600, h]).exp()) for a, b in zip(ends, ends[1:])) * 2.0 ** -30 * float(state[0, h].abs().max())
        assert (off[0, h] <= 2.0 ** -22 * M + 2.0 ** -140).all(), (h, off[0, h].max(), M)
    assert (err <= room + 2.0 ** -18 * want.abs()).all()
    out, final = mcv.gated_delta_rule(*(x.to(cuda) for x in (q, k, 0 * v, g, beta, 0 * state)), normalize=True)
    assert (out == 0).all() and (final == 0).all()


@pytest.mark.parametrize("size", [1.0, 2.0 ** -40])
def test_a_state_that_only_decays(mcv, cuda, size):
    """Over many chunks, by 2^-27 and 2^-54 in all: every chunk's parts have their bits where its state is."""
    q, k, v, g, beta, state = _delta_case(6, [600], 2, 2, 64, 32)
    scale, err, room, off, want, S = _run(mcv, cuda, (q, k, 0 * v, g, beta, size * state), [600])
    # 2^-22 a chunk of a state that its decay, 2^-6 a chunk at most, takes down while its error stays: 2^-16
    assert all(off[0, h].norm() <= 2.0 ** -16 * S[0, h].norm() and S[0, h].norm() > 0 for h in range(2))
