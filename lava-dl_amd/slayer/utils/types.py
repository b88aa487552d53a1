"""Modules whose own tensors keep their type."""
import torch


class KeepsTypes(torch.nn.Module):
    """A module whose own parameters and buffers, and those of the children in ``kept``, keep their type where the module's type is
    changed; the other children follow (``.to(torch.bfloat16)`` makes projections bfloat16, decays stay float32)."""

    kept = ()

    def _apply(self, fn, recurse=True):
        """As torch's, but what has a type of its own keeps it where ``fn`` changes types."""
        def keep(t):
            changed = fn(t)
            return changed if changed.dtype == t.dtype else t.to(changed.device)

        if recurse:
            for name, child in self.named_children():
                child._apply(keep if name in self.kept else fn)
        return super()._apply(keep, recurse=False)
