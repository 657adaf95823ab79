"""The operators together: a recurrent student is distilled, and continues a prompt token by token as it would read it whole."""
import pytest
import torch

from flashlstm_poc_amd.student import RecurrentStudent, successor_teacher, train

pytestmark = pytest.mark.gpu


def test_distilled_student_follows_its_teacher():
    torch.manual_seed(0)
    student = RecurrentStudent(200, 128, 2)
    teacher = successor_teacher(200, 6)
    losses = train(student, teacher, 150, length=32, batch=16)
    assert all(v == v for v in losses) and sum(losses[-10:]) < 0.2 * sum(losses[:10])
    prompt = torch.randint(0, 200, (5, 3), device="cuda")
    out = student.generate(prompt, 12)
    follows = torch.cat([prompt[-1:], out])
    assert float((teacher[1][follows[:-1].long(), 0] == follows[1:]).float().mean()) > 0.9


def test_tokens_one_by_one_and_in_pieces():
    torch.manual_seed(1)
    student = RecurrentStudent(50, 96, 4, layers=2)
    tokens = torch.randint(0, 50, (70, 3), device="cuda")
    with torch.no_grad():
        whole, end = student(tokens)
        first, state = student(tokens[:30])
        rest, state = student(tokens[30:], state)
    # fp16 activations of order one, rounded (2^-11) a dozen times in each of two layers
    assert float((torch.cat([first, rest]).float() - whole.float()).abs().max()) < 0.05
    with torch.no_grad():
        _, state = student(tokens[:1])
    for t in range(1, 70):
        logits, state = student.step(tokens[t], state)
        assert float((logits.float() - whole[t].float()).abs().max()) < 0.05, t
    for a, b in zip(state, end):
        assert torch.allclose(a.memory, b.memory, rtol=0.05, atol=0.05)


def test_refusals():
    with pytest.raises(ValueError, match="multiple"):
        RecurrentStudent(50, 100, 3)


def test_no_tokens_asked_for():
    student = RecurrentStudent(50, 64, 2)
    prompt = torch.randint(0, 50, (4, 3), device="cuda")
    one = student.generate(prompt, 1)
    assert student.generate(prompt, 0).shape == (0, 3) and one.shape == (1, 3)
    assert torch.equal(student.generate(prompt, 5)[:1], one)
