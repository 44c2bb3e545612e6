"""The move-sequence policy: its tokens and records on the CPU, its training
step with this package's operators on the GPU."""
import numpy as np
import pytest
import torch

from alphazero_b200 import host_lib, move_model


@pytest.mark.parametrize("board", [5, 9, 19])
def test_tokens_are_the_moves_between_boards(board):
    planes = host_lib.random_positions(board, 60, 3, 40)
    tokens = move_model.tokens_from_planes(planes, board)
    stones = planes.reshape(60, 17, -1)
    stones = stones[:, :8] + stones[:, 8:16] > 0
    assert tokens.shape == (60, 7) and tokens.min() >= -1 and tokens.max() <= board * board
    for n in range(60):
        for i in range(7):
            now, before, t = stones[n, i], stones[n, i + 1], tokens[n, i]
            if t == -1:
                assert not now.any()
            elif t == board * board:
                assert not (now & ~before).any()
            else:  # one new stone; whatever else changed was captured
                assert now[t] and not before[t] and (now & ~before).sum() == 1


def test_records_are_read(tmp_path):
    rng = np.random.default_rng(0)
    want = [(rng.random(17 * 25).astype("<f4"), rng.random(26).astype("<f4")) for _ in range(5)]
    for f, part in (("game_0.bin", want[:2]), ("game_1.bin", want[2:])):
        with open(tmp_path / f, "wb") as out:
            out.write(np.int32(len(part)).tobytes())
            for state, policy in part:
                for v in (state, policy):
                    out.write(np.int32(v.size).tobytes() + v.tobytes())
                out.write(np.float32(1).tobytes())
    planes, policies = move_model.read_records(str(tmp_path), 5)
    assert np.array_equal(planes, [w[0] for w in want]) and np.array_equal(policies, [w[1] for w in want])
    with pytest.raises(ValueError, match="9x9"):
        move_model.read_records(str(tmp_path), 9)
    with pytest.raises(FileNotFoundError):
        move_model.read_records(str(tmp_path / "none"), 5)


@pytest.mark.gpu
def test_gradients_match_autograd():
    model = move_model.MoveModel(9, dim=32, hidden=64, blocks=2, seed=3)
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(-1, 82, (200, 7), generator=g).cuda()
    targets = torch.randint(-1, 82, (200,), generator=g).cuda()
    loss, got = model.gradients(tokens, targets)
    p = {k: v.double().requires_grad_() for k, v in model.half().items()}
    e = torch.where((tokens >= 0)[..., None], p["table"][tokens.clamp(min=0)], 0.0) * model.scale
    h = torch.nn.functional.gelu(e.flatten(1) @ p["in.w"].t() + p["in.b"])
    for i in range(2):
        h = h + torch.nn.functional.gelu(h @ p[f"{i}.w"].t() + p[f"{i}.b"])
    want = torch.nn.functional.cross_entropy(h @ p["head.w"].t() + p["head.b"], targets, ignore_index=-1)
    want.backward()
    # eight roundings to 8 bits on the longest way from the loss to the table
    assert abs(loss.item() - want.item()) <= 8 * 2.0 ** -8 * want.item()
    for k, v in p.items():
        assert (got[k].double() - v.grad).norm() <= 8 * 2.0 ** -8 * v.grad.norm(), k


@pytest.mark.gpu
def test_training_lowers_the_loss_and_scoring_agrees():
    planes = host_lib.random_positions(9, 512, 4, 60)
    tokens = torch.from_numpy(move_model.tokens_from_planes(planes, 9)).cuda()
    targets = torch.from_numpy(move_model.engine_targets(planes, 9, 0)).cuda()
    model = move_model.MoveModel(9)
    before = model.score(tokens, targets)[0].item()
    for _ in range(40):
        model.step(tokens, targets, 0.2)
    after, rows = model.score(tokens, targets)
    assert after.item() < 0.7 * before
    one = torch.nn.functional.cross_entropy(model.logits(tokens[:1]).double(), targets[:1]).item()
    # the logits are rounded to 8 bits
    assert abs(one - rows[0].item()) <= 2 * 2.0 ** -8 * (one + model.logits(tokens[:1]).abs().max().item())
