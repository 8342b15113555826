from .experts import MoEExperts, MoEExpertsFP8, MoEExpertsSerial, MoEExpertsW4

__all__ = ["MoEExperts", "MoEExpertsSerial", "MoEExpertsFP8", "MoEExpertsW4"]
