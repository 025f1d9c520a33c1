"""torchrun worker for test_e4m3_ranks_cpu: a model of dtype "fp8_w8a8" on several gloo ranks; rank 0 drives, the others follow.  Three prompts, two
decode steps and a short generation; saves rank 0's logits and what each rank holds."""
import os
import sys

import torch
import torch.distributed as dist

import xfastertransformer_b200 as xft

path, out = sys.argv[1], sys.argv[2]
model = xft.AutoModel.from_pretrained(path, dtype="fp8_w8a8")
g = torch.Generator().manual_seed(3)
prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (21, 5, 13)]
two = torch.randint(0, 512, (2, 7), generator=g)
m = model.model
if model.rank == 0:
    sid = model.set_input_cb(prompts, None, 64)
    logits = [model.forward_cb().float()]
    for t in (7, 11):
        model.set_input_cb([[t], [t + 1], [t + 2]], sid, 64)
        logits.append(model.forward_cb().float())
    model.free_seqs(sid)
    tokens = model.generate(two, max_length=10)
else:
    for _ in range(3):
        model.set_input_cb()
        model.forward_cb()
    model.free_seqs()
    model.generate()
d = m.decoder
held = [None] * dist.get_world_size()
experts = next((L for L in d.layers if getattr(L, "experts", None)), None)
dist.all_gather_object(held, dict(
    down=[L.down.in_features if getattr(L, "down", None) is not None else None for L in d.layers], layers=(d.l0, d.l1),
    experts=None if experts is None else (experts.e0, len(experts.experts), [e[1].in_features for e in experts.experts]),
    shared=None if getattr(experts, "shared", None) is None else experts.shared[1].in_features, pairs=m.prefill_decoder.pairs_run,
    sent=m.ctx.stats.get("all_to_all", 0), left=d._pending is not None or m.prefill_decoder._pending is not None))
if model.rank == 0:
    torch.save({"logits": logits, "tokens": tokens, "held": held}, out)
m._closed = True
dist.barrier()
dist.destroy_process_group()
os._exit(0)                                             # gloo: no thread of it outlives the interpreter
