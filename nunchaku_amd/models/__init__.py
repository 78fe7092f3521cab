from .linear import AWQW4A16Linear, SVDQW4A4Linear, W8A8Linear

__all__ = ["SVDQW4A4Linear", "AWQW4A16Linear", "W8A8Linear"]
