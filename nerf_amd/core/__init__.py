from .features import FeatureMapping, FourierFeatures, PositionalEncoding
from .model import NeRF
from .mx4 import Mx4Linear, Mx4NeRF
from .renderer import BoundedVolumeRaymarcher
from .scheduler import IndendityScheduler, LogDecayScheduler, MipNeRFScheduler, Scheduler

__all__ = ["FeatureMapping", "FourierFeatures", "PositionalEncoding", "NeRF", "Mx4Linear", "Mx4NeRF", "BoundedVolumeRaymarcher",
           "IndendityScheduler", "LogDecayScheduler", "MipNeRFScheduler", "Scheduler"]
