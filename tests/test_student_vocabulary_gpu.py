"""The student's vocabulary: its embedding under the names that torch's has, tokens outside it, a teacher of more tokens, and the way that ends at once."""
import pytest
import torch

from flashlstm_poc_amd.student import RecurrentStudent, successor_teacher, train

pytestmark = pytest.mark.gpu


def _student(seed=0):
    torch.manual_seed(seed)
    return RecurrentStudent(60, 96, 4, recurrence="gated")


def test_embedding_has_the_names_of_torchs():
    table, own = torch.nn.Embedding(60, 96), _student().embedding
    assert (own.num_embeddings, own.embedding_dim, own.padding_idx) == (table.num_embeddings, table.embedding_dim, table.padding_idx)


def test_tokens_outside_are_padding():
    student, tokens = _student(), torch.randint(0, 60, (20, 3), device="cuda")
    tokens[4:9], tokens[12, 1] = -1, 60
    assert not bool(student.embedding(tokens)[4:9].any()) and not bool(student.embedding(tokens)[12, 1].any())
    student(tokens)[0].sum().backward()
    assert all(bool(p.grad.isfinite().all()) for p in student.parameters())


def test_a_teacher_of_more_tokens_is_refused():
    student = _student()
    before = student.embedding.weight.detach().clone()
    with pytest.raises(ValueError, match="61 tokens"):
        train(student, successor_teacher(61, 5), 2, length=8, batch=2)
    assert torch.equal(student.embedding.weight, before)
    assert len(train(student, successor_teacher(50, 5), 2, length=8, batch=2)) == 2


def test_the_way_that_ends_at_once_stays_the_best():
    """`end` is the likeliest token behind the prompt: that way's score stays, and all others' start below it and fall."""
    student = _student(4)
    prompt = torch.randint(0, 60, (5, 2), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    with torch.no_grad():
        log_p = torch.log_softmax(student(prompt)[0][-1, 0].double(), -1)
    end = int(log_p.argmax())
    found, scores = student.search(prompt, 10, 6, end=end)
    assert bool((found[0, 0] == end).all())
    # fp16 logits of order one (2^-11 a rounding) come from the same kernels; the score is one rounding of a sum that is off by 48 units of 2^-24
    assert abs(float(scores[0, 0]) - float(log_p[end])) <= 49 * 2.0 ** -24 * max(1.0, abs(float(log_p[end])))
