"""When shared keys are read once for all, and how such a launch is laid out, on the host."""
import random

import torch


def test_blocks_hold_the_rows_of_every_step():
    """As many blocks of rows as the runs can have at most, however their tokens are spread over the requests, and for every replay of a captured step."""
    from tempura_amd.kernels import ops
    rng = random.Random(9)
    for _ in range(2000):
        counts = [rng.choice((1, 2, 7, 40)) for _ in range(rng.choice((1, 2, 9)))]
        lengths = [16 * rng.choice((0, 1, 30, 4000)) for _ in counts]
        shared = ops.SharedKeys(counts, lengths, "cpu")
        if not shared.max_keys:
            continue
        r, kvh, group, longest = sum(counts), rng.choice((1, 2, 8)), rng.choice((1, 3, 4, 8, 34)), rng.choice((1, 2, 30, 400))
        new = [rng.choice((1, longest, rng.randint(1, longest))) for _ in range(r)]
        plan = ops._prefix_plan(shared, r, sum(new), group, kvh, longest, rng.choice((256, 4096)), rng.choice((32, 64, 128)), rng.choice((torch.bfloat16, torch.float32)))
        at, need = 0, 0
        for c, v in zip(counts, lengths):
            need += -(-sum(new[at: at + c]) * group // plan[0]) if v else 0
            at += c
        assert plan[2] >= need


def test_blocks_hold_the_rows_of_every_replay():
    from tempura_amd.kernels import ops
    rng = random.Random(10)
    for _ in range(2000):
        groups, r, group = rng.choice((3, 5, 9, 17)), rng.choice((2, 8, 64, 200)), rng.choice((1, 3, 4, 8, 34))
        data = torch.zeros(2 * groups + 1 + r, dtype=torch.int32)
        shared = ops.SharedKeys.captured(data, r, groups, 16 * rng.choice((16, 64, 512)))
        plan = ops._prefix_plan(shared, r, r, group, rng.choice((1, 2, 8)), 1, 512, 128, torch.bfloat16)
        runs, left = [], r
        for _ in range(rng.randint(1, ops.SharedKeys.runs_in(groups))):
            if left:
                runs.append((rng.randint(1, left), 16 * rng.randint(1, shared.max_keys // 16)))
                left -= runs[-1][0]
        out = data.numpy()
        ops.SharedKeys.pack(runs, r, groups, out)
        assert plan[2] >= sum(-(-(int(shared.starts[g + 1]) - int(shared.starts[g])) * group // plan[0]) for g in range(groups) if int(shared.keys[g]))
        assert plan[3] * plan[4] * 32 >= shared.max_keys
