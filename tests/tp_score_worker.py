"""Worker of test_token_loss_more_cpu.py (under ``torch.distributed.run``, gloo): scores, and the losses that read them, of a model
under tensor parallelism, whose ranks see their shares of a chunk's positions, against the unsharded model."""
import json
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from parallel_engine_worker import RAGGED, build, ft  # noqa: E402
from flextrain_b200.nn.loss import DistillationLoss, PolicyLoss  # noqa: E402


class Staged:
    """Gathers as over peer memory: into one buffer for each size."""

    def __init__(self, tp):
        self.tp, self.stage = tp, {}

    def __getattr__(self, name):
        return getattr(self.tp, name)

    def all_gather(self, x):
        full = self.tp.all_gather(x)
        nb = full.numel() * full.element_size()
        stage = self.stage.setdefault(nb, torch.empty(nb, dtype=torch.uint8))
        stage.copy_(full.view(-1).view(torch.uint8))
        return stage.view(full.dtype).view(full.shape)


def sequences(K=None):
    seqs = ft.SyntheticTokenSource(512, RAGGED, seed=5).get_sequences(sum(RAGGED))
    g = torch.Generator().manual_seed(3)
    for s in seqs:
        n = len(s)
        s.advantages = torch.randn(n, generator=g)
        if K:
            s.old_logprobs, s.ref_logprobs = -6 - torch.rand(n, generator=g), -6 - torch.rand(n, generator=g)
            s.teacher_ids = torch.randint(0, 512, (n, K), generator=g)
            s.teacher_logprobs = torch.log_softmax(torch.randn(n, K, generator=g), -1)
    return seqs


def results(am):
    out = {}
    for K in (1, 4):
        for i, x in enumerate(am.score(sequences(), top_k=K, temperature=0.8)):
            for name, v in x._asdict().items():
                out[f"{K}/{i}/{name}"] = v
    for name, loss in (("policy", PolicyLoss(kl_coef=0.1, entropy_coef=0.01)), ("distill", DistillationLoss(rest="bucket", ce_weight=0.2))):
        seqs = sequences(K=3)
        am.evaluate(seqs, loss_fn=loss)
        for i, s in enumerate(seqs):
            out[f"{name}/{i}"] = s.per_token_loss
    return out


def main():
    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    dist.init_process_group("gloo")
    am = build("cpu", torch.float32, world, rank, "tp_ragged", "collective")
    am.tp = Staged(am.tp)
    got = results(am)
    if rank == 0:
        want = results(build("cpu", torch.float32, 1, 0, "tp_ragged", "collective"))
        worst, ids = 0.0, 0
        for k, v in want.items():
            if v.dtype == torch.int64:
                ids += int((v != got[k]).sum())
            else:
                worst = max(worst, float((v - got[k]).abs().max()))
        with open(sys.argv[1], "w") as f:
            json.dump({"worst": worst, "ids": ids, "fields": len(want), "ids_of": sum(v.numel() for v in want.values() if v.dtype == torch.int64)}, f)
    dist.barrier()
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
