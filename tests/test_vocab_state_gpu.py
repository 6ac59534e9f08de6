"""What a loss of the vocabulary head hands back, keeps and needs on the device: a loss that may be changed in place, a
state that a backward leaves as it was, workspaces within their bound, the launches that are counted, and results that
say so when a kernel gave up a wait."""
import pytest
import torch

from predicitivecoding_b200 import ops
from predicitivecoding_b200.ops import vocab
from test_vocab_gpu import head, teacher

pytestmark = pytest.mark.gpu
DEV = "cuda"
STATUS = 4          # word of the state's counters


def counters(state):
    """The state's int32 words: counted rows, blocks done, K splits of dw and dx, status of a wait."""
    at = state.N * ((state.D + 7) // 8 * 8) * 2
    return state.saved.view(torch.int32)[(at + 255) // 256 * 64:][:8]


def forms(N, V, D, seed=3):
    x, w, tgt, g = head(N, V, D, seed)
    ids, t = teacher(N, V, 6, tgt, g, torch.float32)
    return x, w, {"ce": lambda x, w, r="mean": vocab.ce_fwd(x, w, tgt, -1, r),
                  "distill": lambda x, w, r="mean": vocab.distill_fwd(x, w, ids, t, 2.0, r)}, \
        {"ce": lambda x, w, r="mean": vocab.cross_entropy(x, w, tgt, -1, r),
         "distill": lambda x, w, r="mean": vocab.distill(x, w, ids, t, 2.0, r)}


@pytest.mark.parametrize("N,V", [(3, 900), (300, 900), (300, 200)])
@pytest.mark.parametrize("kind", ["ce", "distill"])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_a_loss_may_be_changed_in_place(N, V, kind, reduction):
    x, w, fwd, auto = forms(N, V, 64)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = auto[kind](xg, wg, reduction)
    whole = float(loss.detach())
    loss /= 4
    assert float(loss.detach()) == whole / 4
    loss.backward()
    first, state = fwd[kind](x, w, reduction)
    dx, dw = vocab.head_bwd(state, 0.25)
    assert torch.equal(xg.grad, dx) and torch.equal(wg.grad, dw)
    first.zero_()                                  # the gradient does not read it again
    again = vocab.head_bwd(state, 0.25)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("N,V,D", [(3, 5000, 64), (40, 5000, 64), (300, 5000, 64), (200, 2000, 1024), (300, 300, 64)])
@pytest.mark.parametrize("kind", ["ce", "distill"])
def test_a_backward_leaves_the_state_as_it_was(N, V, D, kind):
    """Two backwards of one state may run at the same time, in pieces of different sizes."""
    x, w, fwd, _ = forms(N, V, D)
    _, state = fwd[kind](x, w)
    if V > 512:
        counters(state)[2:4] = -7                  # the splits are each backward's own
    before = state.saved.clone()
    pieces = (0, 256, 1024, 2560)
    want = [vocab.head_bwd(state, piece=p) for p in pieces]
    assert torch.equal(state.saved, before)
    side = [torch.cuda.Stream() for _ in pieces]
    got = []
    for s, p in zip(side, pieces):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(vocab.head_bwd(state, piece=p))
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("N,V", [(1, 300000), (200, 300000), (300, 262144), (257, 270001)])
def test_the_workspace_of_g_is_bounded(N, V):
    """256 MiB of g by default, however many rows its panels are padded to."""
    x, w, tgt, _ = head(N, V, 16, 4)
    _, state = vocab.ce_fwd(x, w, tgt)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    dw = vocab.head_bwd(state, need_dx=False)[1]
    torch.cuda.synchronize()
    extra = torch.cuda.max_memory_allocated() - held - dw.numel() * 2
    assert extra <= (256 << 20) + (1 << 20)


def launches(f):
    before = ops.launch_count()
    f()
    return ops.launch_count() - before


def test_launches_are_counted():
    """Lists are sorted (1), long batches counted (1), rows packed (1), logits (1), row losses (1); loss and g of whole
    vocabularies come of one launch; rows of w that no vector fits are copied (1).  A backward: g and both
    products for each piece, and the gather."""
    for N, long in ((8192, 0), (8193, 1)):
        for V, whole in ((512, 1), (700, 0)):
            x, w, fwd, _ = forms(N, V, 16)
            apart = torch.zeros(V, 21, device=DEV, dtype=torch.bfloat16)[:, 2:18].copy_(w)
            for kind, lists in (("ce", 0), ("distill", 1)):
                made = lists + long + 1 + (1 if whole else 2)
                assert launches(lambda: fwd[kind](x, w)) == made
                assert launches(lambda: fwd[kind](x, apart)) == made + 1
                assert launches(lambda: fwd[kind](x, w, "none")) == lists + long + 3
                state = fwd[kind](x, w)[1]
                assert launches(lambda: vocab.head_bwd(state)) == (1 if whole else 2) + 1
                if not whole:
                    assert launches(lambda: vocab.head_bwd(state, piece=256)) == 2 * 3 + 1
                    assert launches(lambda: vocab.head_bwd(state, need_dx=False)) == 3


@pytest.mark.parametrize("N,V,D", [(3, 700, 64), (40, 700, 64), (300, 5000, 64), (200, 2000, 1024), (300, 300, 64),
                                   (700, 30000, 264)])
@pytest.mark.parametrize("f32", [False, True])
def test_gradients_behind_a_wait_that_ran_out_are_nan(N, V, D, f32):
    """A kernel that gives up a wait records it in the state and leaves its outputs unfinished: the gradients are NaN
    then, whichever launch writes them, so nobody trains on them."""
    x, w, fwd, _ = forms(N, V, D)
    _, state = fwd["ce"](x, w)
    assert state.status() == 0
    counters(state)[STATUS] = 2
    assert state.status() == 2
    dt = torch.float32 if f32 else torch.bfloat16
    new = lambda *s: torch.zeros(*s, device=DEV, dtype=dt)
    nan = lambda t: bool(torch.isnan(t.float()).all())
    for piece in (0, 512):
        dx, dw = vocab.head_bwd(state, dx=new(N, D), dw=new(V, D), piece=piece)
        assert nan(dx) and nan(dw)
        assert nan(vocab.head_bwd(state, dx=new(N, D), need_dw=False, piece=piece)[0])
        assert nan(vocab.head_bwd(state, dw=new(V, D), need_dx=False, piece=piece)[1])
        assert nan(vocab.head_bwd(state, dw=new(V, D), accumulate=True, piece=piece)[1])
    apart = new(N, D + 16)[:, 8:8 + D]
    rows = new(V, D + 5)[:, 3:3 + D]
    vocab.head_bwd(state, dx=apart, dw=rows)
    assert nan(apart) and nan(rows)
    counters(state)[STATUS] = 0
    assert not bool(torch.isnan(vocab.head_bwd(state)[1].float()).any())


@pytest.mark.parametrize("temperature", [0.0, -1.0, float("inf"), float("nan"), 1e-60, 1e60])
def test_what_is_no_temperature_in_32_bits_is_refused(temperature):
    x, w, tgt, g = head(8, 40, 16, 15)
    ids, t = teacher(8, 40, 4, tgt, g, torch.float32)
    with pytest.raises(ValueError):
        vocab.distill_fwd(x, w, ids, t, temperature)
