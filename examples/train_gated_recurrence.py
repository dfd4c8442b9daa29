"""A DTDG model whose temporal part is a stack of gated recurrent blocks instead of a cell
per snapshot: the Flare pipeline's windows feed a two-layer GCN, the window's rows go
through ``GatedRecurrentStack`` at once (scan, fused norms, 8-bit saved activations), and
evaluation advances the blocks one snapshot at a time on a table of states.

    python examples/train_gated_recurrence.py --device cuda
    python examples/train_gated_recurrence.py --nodes 2000 --edges 20000 --snapshots 16 --device cpu
    python examples/train_gated_recurrence.py --device cuda --checkpoint none --epochs 5

The session prepares the data, slides the windows and runs the steps; only its model and
optimizer are replaced. ``--checkpoint int8`` (the default) keeps the activations that the
blocks save in 8 bits, and ``saved8`` does the same for the GCN's and the linear layers'.
On CUDA every training window is one captured graph, as for the built-in models.
"""
from __future__ import annotations

import argparse
import sys
from contextlib import nullcontext
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch
from torch import nn

from starry_unigraph.lib_stable import GatedRecurrentStack, GCNStack, saved8
from starry_unigraph.ops.dtdg import linear


class GatedRecurrenceModel(nn.Module):
    def __init__(self, input_size: int, hidden_size: int, output_size: int = 1, checkpoint: str | None = None):
        super().__init__()
        self.checkpoint = checkpoint
        self.gcn = GCNStack(input_size, hidden_size, num_layers=2)
        self.blocks = GatedRecurrentStack(hidden_size, num_layers=2, checkpoint=checkpoint)
        self.out = nn.Linear(hidden_size, output_size)

    def forward(self, blob_or_graph, state=None):
        single = hasattr(blob_or_graph, "edge_src")
        with saved8() if self.checkpoint else nullcontext():
            feats = self.gcn.layerwise(blob_or_graph)
            if single and not torch.is_grad_enabled():  # one snapshot: advance the states in place
                if state is None:
                    state = self.blocks.init_state(feats[0].size(0))
                n = self.blocks.step(feats[0], state)
                return linear(n, self.out.weight, self.out.bias), state
            n, state = self.blocks(torch.stack(feats), state)
            preds = [linear(rows, self.out.weight, self.out.bias) for rows in n]
        return (preds[-1] if single else preds), state


def main(argv=None) -> dict:
    from starry_unigraph import SchedulerSession
    from starry_unigraph.backends.dtdg.runtime.training import FlareOptimizer

    root = Path(__file__).resolve().parents[1]
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--config", default=str(root / "configs" / "mpnn_lstm_nvlink.yaml"))
    p.add_argument("--nodes", type=int, default=20_000)
    p.add_argument("--edges", type=int, default=200_000)
    p.add_argument("--snapshots", type=int, default=32)
    p.add_argument("--epochs", type=int, default=3)
    p.add_argument("--device", default="cpu")
    p.add_argument("--checkpoint", default="int8", choices=["int8", "none"])
    p.add_argument("--artifact-root", default=None)
    a = p.parse_args(argv)
    s = SchedulerSession.from_config(a.config, overrides={
        "runtime": {"device": a.device}, "train": {"epochs": a.epochs, "snaps": a.snapshots},
        "data": {"synthetic": {"num_nodes": a.nodes, "edges_per_snapshot": a.edges, "num_snapshots": a.snapshots}}})
    if a.artifact_root:
        s.ctx.artifact_root = Path(a.artifact_root)
    s.prepare_data()
    s.build_runtime()
    built = s.runtime.state["flare_model"]
    torch.manual_seed(int(s.ctx.config["train"].get("seed", 0)))
    model = GatedRecurrenceModel(built["input_size"], built["hidden_size"], built["output_size"],
                                 None if a.checkpoint == "none" else a.checkpoint).to(a.device)
    s.runtime.model = model
    s.runtime.optimizer = FlareOptimizer(model, float(s.ctx.config["train"]["lr"]), torch.device(a.device))
    result: dict = {"train": [], "val": []}
    for epoch in range(a.epochs):
        tr, va = s.run_epoch("train"), s.run_epoch("val")
        print(f"epoch {epoch + 1} | train loss {tr['global_loss']:.5f} | val loss {va['global_loss']:.5f}", flush=True)
        result["train"].append(tr["global_loss"])
        result["val"].append(va["global_loss"])
    result["test"] = len(s.predict("test").predictions)
    return result


if __name__ == "__main__":
    main()
