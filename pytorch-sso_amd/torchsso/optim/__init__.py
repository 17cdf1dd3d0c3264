from torchsso.optim.secondorder import SecondOrderOptimizer  # NOQA
from torchsso.optim.vi import VIOptimizer, VOGN  # NOQA
from torchsso.optim.muon import Muon, muon  # NOQA
from torchsso.optim.adamw import AdamW, adamw, adamw_states  # NOQA
from torchsso.optim import lr_scheduler  # NOQA
