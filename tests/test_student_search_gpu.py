"""The operators together: a student with a gated recurrence, its gradients, its tokens one by one, and the search with beams."""
import pytest
import torch

from flashlstm_poc_amd.student import RecurrentStudent, successor_teacher, train
from lm_helpers import U32

pytestmark = pytest.mark.gpu


def _tokens(vocabulary, *shape, seed=0):
    return torch.randint(0, vocabulary, shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _student(recurrence, seed=0, **more):
    torch.manual_seed(seed)
    return RecurrentStudent(60, 96, 4, recurrence=recurrence, **more)


def test_trains_with_a_gated_recurrence():
    losses = train(_student("gated", layers=2), successor_teacher(60, 5), 3, length=40, batch=6)
    assert len(losses) == 3 and all(v == v and v > 0 for v in losses)


@pytest.mark.parametrize("recurrence", ["lstm", "gated"])
def test_embedding_gradient_is_the_table_rows_sum(recurrence):
    """The student's gradients with its own embedding and with rows gathered by indexing, whose gradient torch adds up: the same fp16 rows, added in 32
    bits in another order, k - 1 additions each for a token that occurs k times, off by at most u of the sum of magnitudes."""
    student, tokens = _student(recurrence), _tokens(60, 50, 4)
    d = torch.randn(50, 4, 60, device="cuda").half()
    student(tokens)[0].backward(d)
    grads = {n: p.grad.clone() for n, p in student.named_parameters()}
    assert all(bool(g.isfinite().all()) and bool(g.any()) for g in grads.values())
    student.zero_grad(set_to_none=True)
    rows = student.embedding.weight.detach()[tokens].half().requires_grad_()
    stream, added = rows, None
    for layer in student.layers:
        stream, added, _ = layer(stream, added, None)
    student._logits(stream, added).backward(d)
    for name, p in student.named_parameters():
        if name != "embedding.weight":
            assert torch.equal(p.grad, grads[name]), name
    sums = lambda x: torch.zeros(60, x.shape[1], device="cuda", dtype=torch.float64).index_add_(0, tokens.flatten(), x)
    flat = rows.grad.flatten(0, 1).double()
    count = torch.bincount(tokens.flatten(), minlength=60)[:, None]
    assert bool(((grads["embedding.weight"].double() - sums(flat)).abs() <= U32 * (count + 1) * sums(flat.abs())).all())


def test_gated_tokens_one_by_one_and_in_pieces():
    student, tokens = _student("gated", 1, layers=2), _tokens(60, 300, 3, seed=1)
    with torch.no_grad():
        whole, end = student(tokens)
        first, state = student(tokens[:130])
        rest, state = student(tokens[130:], state)
        # fp16 activations of order one, rounded (2^-11) a dozen times in each of two layers
        assert float((torch.cat([first, rest]).float() - whole.float()).abs().max()) < 0.05
        _, state = student(tokens[:280])
    for t in range(280, 300):
        logits, state = student.step(tokens[t], state)
        assert float((logits.float() - whole[t].float()).abs().max()) < 0.05, t
    for a, b in zip(state, end):
        assert a.h is None and torch.allclose(a.c, b.c, atol=0.05) and torch.allclose(a.memory, b.memory, rtol=0.05, atol=0.05)


def _score(student, prompt, found):
    """The logarithm of a continuation's probability, (B,), by one pass over prompt and continuation (count, B)."""
    with torch.no_grad():
        logits, _ = student(torch.cat([prompt, found[:-1]]))
    log_p = torch.log_softmax(logits[len(prompt) - 1:].double(), -1)
    return log_p.gather(-1, found[..., None])[..., 0]


@pytest.mark.parametrize("recurrence", ["lstm", "gated"])
def test_search_scores_are_those_of_its_ways(recurrence):
    student, prompt = _student(recurrence, 2), _tokens(60, 7, 3, seed=2)
    found, scores = student.search(prompt, 9, 4)
    assert found.shape == (3, 4, 9) and bool((scores[:, :-1] >= scores[:, 1:]).all()) and bool((found >= 0).all())
    for k in range(4):
        # nine steps, whose logits are off as above in single tokens
        assert float((_score(student, prompt, found[:, k].t().contiguous()).sum(0) - scores[:, k]).abs().max()) < 9 * 0.05
    for a in range(4):
        for b in range(a):
            assert not bool((found[:, a] == found[:, b]).all(-1).any())     # no way twice
    again = student.search(prompt, 9, 4)
    assert torch.equal(again[0], found) and torch.equal(again[1], scores)


@pytest.mark.parametrize("recurrence", ["lstm", "gated"])
def test_one_beam_is_the_likeliest_token(recurrence):
    student, prompt = _student(recurrence, 3), _tokens(60, 5, 2, seed=3)
    assert torch.equal(student.search(prompt, 8, 1)[0][:, 0].t(), student.generate(prompt, 8))
    assert student.search(prompt, 0, 3)[0].shape == (2, 3, 0)
    one = student.search(prompt, 1, 5)
    with torch.no_grad():
        want = torch.sort(torch.log_softmax(student(prompt)[0][-1].double(), -1), dim=-1, descending=True, stable=True)
    assert torch.equal(one[0][..., 0], want.indices[:, :5])


def test_ways_that_end():
    student, prompt = _student("gated", 4), _tokens(60, 5, 2, seed=4)
    end = int(student.generate(prompt, 1)[0, 0])
    found, scores = student.search(prompt, 10, 6, end=end)
    ended = (found == end).int().cummax(-1).values.bool()
    assert bool((found[ended] == end).all()) and bool(ended.any()) and bool(scores.isfinite().all())
    first = found[0, :, 0] == end                                            # the way that ends at once: its score is its one token's
    log_p = torch.log_softmax(student(prompt)[0][-1, 0].double(), -1)[end]
    if bool(first.any()):
        assert abs(float(scores[0][first][0]) - float(log_p)) < 1e-3


def test_more_beams_than_tokens():
    torch.manual_seed(5)
    student, prompt = RecurrentStudent(3, 64, 2, recurrence="gated"), _tokens(3, 4, 2, seed=5)
    found, scores = student.search(prompt, 2, 8)
    assert bool((scores.isfinite() == (found[..., 1] >= 0)).all()) and bool(scores[:, :8].isfinite().all())    # 9 ways of two tokens
    found, scores = student.search(prompt, 1, 8)
    assert bool(scores[:, :3].isfinite().all()) and bool((found[:, 3:] == -1).all()) and not bool(scores[:, 3:].isfinite().any())


def test_refusals():
    with pytest.raises(ValueError, match="recurrence"):
        RecurrentStudent(50, 64, 2, recurrence="rnn")
    with pytest.raises(ValueError, match="between"):
        RecurrentStudent(50, 64, 2, recurrence="gated").search(_tokens(50, 3, 1), 2, 33)
